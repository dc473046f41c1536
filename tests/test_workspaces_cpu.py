"""CPU test of the general forms' scratch memory: the library's calls release the interpreter lock and take several launches, so two
threads that submit to one stream must not bring the same memory.  The library's entry points are stood in for here: nothing is
launched, and host tensors do."""
import contextlib
import threading

import pytest
import torch

from gnnhwc import _cabi, custom_gn, rotary_frequencies, tokens

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def on_the_host(monkeypatch):
    for module in (custom_gn, tokens):
        monkeypatch.setattr(module, "_check_device", lambda *a: None)
        monkeypatch.setattr(module, "_current_stream_ptr", lambda device: 0)
        monkeypatch.setattr(module, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def _calls():
    x, w = torch.ones(700, 640, dtype=BF16), torch.ones(640)
    q, p, f, qw = torch.ones(2, 30, 4, 64, dtype=BF16), torch.arange(30).view(-1, 1), rotary_frequencies((32,)), torch.ones(64)
    image, affine, stats = torch.ones(2, 600, 64).transpose(1, 2), torch.ones(64), torch.ones(2, 8)
    return {
        "gnnhwc_rms_bwd": lambda: tokens._rms_norm_bwd(x, None, x, w, 1e-6),
        "gnnhwc_rotary_bwd": lambda: tokens._rotary_bwd(q, None, q, None, p, f, [32], False, qw, None, 1e-6),
        "gnnhwc_clip": lambda: tokens._clip_general([x], None, 1.0, 1.0, 1e-6),
        "gnnhwc_fwd_cast": lambda: custom_gn.gn_nhwc_fwd(image, affine, affine, 8, 1e-5, 0),
        "gnnhwc_bwd_cast": lambda: custom_gn.gn_nhwc_bwd(image, image, affine, affine, stats, stats, 8, 0),
    }


@pytest.mark.parametrize("entry", sorted(_calls()))
def test_two_threads_bring_two_workspaces(entry, on_the_host, monkeypatch):
    call, both, seen, failures = _calls()[entry], threading.Barrier(2, timeout=60), [], []

    def meet(*args):
        workspace, size, _stream = args[-3:]
        seen.append((workspace, size))
        both.wait()  # both calls are in the library now, and hold what they brought
        return 0

    def run():
        try:
            call()
        except BaseException as e:  # (for the test's own thread)
            failures.append(e)

    monkeypatch.setattr(_cabi.lib, entry, lambda *args: 0)
    call()  # whatever is kept between calls is there
    monkeypatch.setattr(_cabi.lib, entry, meet)
    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
    (a, a_size), (b, b_size) = sorted(seen)
    assert a + a_size <= b, entry
