"""CPU checks of attention and dropout: argument blocks, refusals before anything is launched, workspaces, the Python surface
without a device, and the generator against its published vectors."""
import ctypes
import math
import os

import numpy as np
import pytest
import torch

import gnnhwc
from gnnhwc import Dropout, _cabi, dropout, window_attention, window_attention_cached
from tests.dropout_refs import philox

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
lib = _cabi.lib
F32, F64, F16, BF16 = 0, 1, 2, 3


def test_the_argument_block_has_the_headers_layout(tmp_path):
    fields = [f[0] for f in _cabi.WindowCall._fields_]
    source = tmp_path / "layout.c"
    source.write_text('#include <stdio.h>\n#include "gnnhwc_tokens.h"\nint main(void) {\n' + "".join(
        '  printf("%%zu\\n", offsetof(gnnhwc_window_call, %s));\n' % f for f in fields) + '  printf("%zu\\n", sizeof(gnnhwc_window_call));\n  return 0;\n}\n')
    program = tmp_path / "layout"
    assert os.system("gcc -std=c11 -Wall -Werror -include stddef.h -I%s %s -o %s" % (os.path.join(ROOT, "include"), source, program)) == 0
    got = [int(v) for v in os.popen(str(program)).read().split()]
    assert got == [getattr(_cabi.WindowCall, f).offset for f in fields] + [ctypes.sizeof(_cabi.WindowCall)]


def _block():
    raw = ctypes.create_string_buffer(128)
    return raw, (ctypes.addressof(raw) + 15) // 16 * 16


def _call(**change):
    c = _cabi.WindowCall()
    raw, at = _block()
    for n in ("q", "k", "v", "out", "lse", "out_grad", "q_grad", "k_grad", "v_grad"):
        setattr(c, n, at)
    for n in ("q", "k", "v", "out", "out_grad", "q_grad", "k_grad", "v_grad"):
        getattr(c, n + "_stride")[:] = [4096, 256, 64]
    c.batch, c.tokens, c.keys, c.heads, c.kv_heads, c.head_dim, c.window, c.sinks, c.scale, c.dtype = 2, 8, 8, 4, 2, 64, 3, 1, 0.125, BF16
    for n, v in change.items():
        if n.endswith("_stride"):
            getattr(c, n)[:] = v
        else:
            setattr(c, n, at + 8 if v == "odd" else v)
    return c, raw


REFUSED = [(dict(dtype=F64), "dtype"), (dict(dtype=7), "dtype"), (dict(head_dim=0), "head_dim"), (dict(head_dim=12), "head_dim"), (dict(head_dim=264), "head_dim"), (dict(head_dim=136, dtype=F32), "head_dim"),
           (dict(heads=3), "heads"), (dict(kv_heads=0), "heads"), (dict(heads=65536, kv_heads=1), "heads"), (dict(batch=-1), "negative"), (dict(tokens=-1), "negative"),
           (dict(keys=-1, tokens=0), "negative"), (dict(keys=2 ** 30 + 1), "2\\^30"), (dict(window=-2), "window"), (dict(sinks=-1), "sinks"), (dict(tokens=9), "more queries"),
           (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=1e-60), "scale"),
           (dict(length_type=2), "length_type"), (dict(q=None), "q is null"), (dict(v=None), "v is null"), (dict(k="odd"), "aligned"), (dict(out="odd"), "aligned"),
           (dict(q_stride=[4096, 257, 64]), "16 bytes"), (dict(k_stride=[4096, 2 ** 30, 64]), "2\\^25"), (dict(v_stride=[4096, -256, 64]), "stride"),
           (dict(batch=2 ** 20, heads=64, kv_heads=64), "too many"), (dict(batch=2 ** 18, heads=32, kv_heads=32), "too many"), (dict(out_rest="odd"), "out_rest")]


@pytest.mark.parametrize("change,text", REFUSED)
def test_attention_refuses(change, text):
    import re

    c, _keep = _call(**change)
    _raw, ws = _block()
    for run in (lib.gnnhwc_window, lib.gnnhwc_window_bwd):
        assert run(ctypes.byref(c), ws, 1 << 40, None) == -1 and re.search(text, _cabi.last_error()), _cabi.last_error()
    assert lib.gnnhwc_window_workspace_bytes(ctypes.byref(c)) == 0 and lib.gnnhwc_window_bwd_workspace_bytes(ctypes.byref(c)) == 0


def test_workspaces_and_backward_refuse():
    c, _keep = _call()
    assert lib.gnnhwc_window_workspace_bytes(ctypes.byref(c)) == 256  # one workgroup a head: none is needed
    c, _keep = _call(batch=1, keys=5000, window=-1)  # several share a head's keys
    assert lib.gnnhwc_window_workspace_bytes(ctypes.byref(c)) > 256
    assert lib.gnnhwc_window(ctypes.byref(c), None, 1 << 40, None) == -2 and "workspace" in _cabi.last_error()
    assert lib.gnnhwc_window(ctypes.byref(c), _block()[1], 256, None) == -2
    c, _keep = _call()
    small = lib.gnnhwc_window_bwd_workspace_bytes(ctypes.byref(c))
    _raw, ws = _block()
    assert small > 0 and lib.gnnhwc_window_bwd(ctypes.byref(c), ws, small - 1, None) == -2 and lib.gnnhwc_window_bwd(ctypes.byref(c), ws + 8, 1 << 40, None) == -2
    for change, text in ((dict(at_end=1), "cache"), (dict(lse=None), "lse"), (dict(out_grad=None), "out_grad"), (dict(k_grad="odd"), "aligned")):
        c, _keep = _call(**change)
        assert lib.gnnhwc_window_bwd(ctypes.byref(c), ws, 1 << 40, None) == -1 and text in _cabi.last_error()
    c, _keep = _call(batch=2 ** 12, heads=64, kv_heads=64, keys=200, window=3, sinks=100)
    assert lib.gnnhwc_window_workspace_bytes(ctypes.byref(c)) > 0
    assert lib.gnnhwc_window_bwd(ctypes.byref(c), ws, 1 << 60, None) == -1 and "too many" in _cabi.last_error()
    # a batch of nothing launches nothing
    c, _keep = _call(batch=0)
    assert lib.gnnhwc_window(ctypes.byref(c), ws, 1 << 20, None) == 0 and lib.gnnhwc_window_bwd(ctypes.byref(c), ws, 1 << 40, None) == 0
    assert lib.gnnhwc_window(None, ws, 1 << 20, None) == -1


def test_dropout_refuses():
    p = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)
    for args, text in (((p, None, p, 8, -0.1, 0, None, 0, F32), "p must"), ((p, None, p, 8, math.nan, 0, None, 0, F32), "p must"), ((p, None, p, 8, 0.5, 0, None, 0, 9), "dtype"),
                       ((p, None, p, -1, 0.5, 0, None, 0, F32), "size"), ((p, None, p, 2 ** 34 + 1, 0.5, 0, None, 0, F32), "size"), ((None, None, p, 8, 0.5, 0, None, 0, F32), "null"),
                       ((p, None, None, 8, 0.5, 0, None, 0, F32), "null"), ((p, None, p, 8, 0.5, 0, p.value // 8 * 8 + 4, 0, F32), "seed_at")):
        assert lib.gnnhwc_dropout(*args, None) == -1 and text in _cabi.last_error(), _cabi.last_error()
    assert lib.gnnhwc_dropout(None, None, None, 0, 0.5, 0, None, 0, F32, None) == 0


def test_host_tensors_and_bad_shapes_are_refused():
    q = torch.zeros(1, 4, 2, 8)
    for call in (lambda: window_attention(q, q, q), lambda: window_attention_cached(q, q, q, torch.tensor([4])), lambda: dropout(q, 0.5, 1), lambda: Dropout()(q)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="window"):
        window_attention(q, q, q, window=-1)


def test_meta_kernels():
    q, k = torch.zeros((2, 3, 4, 64), device="meta", dtype=torch.bfloat16), torch.zeros((2, 5, 2, 64), device="meta", dtype=torch.bfloat16)
    out, lse, rest = torch.ops.gnop.window_attention(q, k, k, None, 4, 1, True, False, 0.125, True)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (2, 4, 3) and lse.dtype == torch.float32
    assert torch.ops.gnop.window_attention(q, k, k, None, 4, 1, True, True, 0.125, False)[1].numel() == 0
    dq, dk, dv = torch.ops.gnop.window_attention_bwd(out, q, k, k, out, lse, rest, None, 4, 1, True, 0.125)
    assert dq.shape == q.shape and dk.shape == dv.shape == k.shape
    assert torch.ops.gnop.dropout(q, None, 0.1, 1, None, 0).shape == q.shape


def test_dropout_module():
    assert isinstance(Dropout(0.3), torch.nn.Dropout) and not Dropout().state_dict() and "channel_dim=1" in repr(Dropout(0.1, 1))
    x = torch.ones(3)
    assert torch.equal(Dropout(0.3).eval()(x), x) and torch.equal(Dropout(0.0)(x, x), x + x)
    with pytest.raises(ValueError):
        Dropout(1.5)


def test_generator_against_published_vectors():
    """Philox 4x32 of zeros, of ones and of the digits of pi, 10 rounds, as its authors list them."""
    def run(counter, key, rounds):
        return [int(v) for v in philox([np.array(c, dtype=np.uint64) for c in counter], key, rounds)]

    assert run((0, 0, 0, 0), (0, 0), 10) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert run((ones,) * 4, (ones, ones), 10) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert run((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), 10) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    assert run((0, 0, 0, 0), (0, 0), 7) == [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]


def test_the_package_exports_them():
    assert {"window_attention", "window_attention_cached", "dropout", "Dropout"} <= set(dir(gnnhwc))
