"""CPU checks of the operators for token streams: the library exports what include/gnnhwc_tokens.h declares, bad arguments are
refused before anything is launched, workspaces have their sizes, and the Python surface traces without a device."""
import ctypes
import math
import os
import re

import pytest
import torch

import gnnhwc
from gnnhwc import RMSNorm, Rotary, _cabi, rms_norm, rms_norm_quant, rotary, rotary_frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
lib = _cabi.lib
F32, F64, F16, BF16 = 0, 1, 2, 3


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "gnnhwc_tokens.h")).read(), flags=re.S)
    names = set(re.findall(r"\b(gnnhwc_[a-z_0-9]+)\s*\(", text))
    assert {"gnnhwc_rms_fwd", "gnnhwc_rms_fwd_quant", "gnnhwc_rms_bwd", "gnnhwc_rotary", "gnnhwc_rotary_bwd", "gnnhwc_clip"} <= names
    assert names <= set(_cabi.SYMBOLS)


def test_the_argument_block_has_the_headers_layout(tmp_path):
    fields = [f[0] for f in _cabi.RotaryCall._fields_]
    source = tmp_path / "layout.c"
    source.write_text('#include <stdio.h>\n#include "gnnhwc_tokens.h"\nint main(void) {\n' + "".join(
        '  printf("%%zu\\n", offsetof(gnnhwc_rotary_call, %s));\n' % f for f in fields) + '  printf("%zu\\n", sizeof(gnnhwc_rotary_call));\n  return 0;\n}\n')
    program = tmp_path / "layout"
    assert os.system("gcc -std=c11 -Wall -Werror -I%s %s -o %s" % (os.path.join(ROOT, "include"), source, program)) == 0
    got = [int(v) for v in os.popen(str(program)).read().split()]
    assert got == [getattr(_cabi.RotaryCall, f).offset for f in fields] + [ctypes.sizeof(_cabi.RotaryCall)]


def _p():
    return ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p)


@pytest.mark.parametrize("change,text", [(dict(C=0), "channels"), (dict(C=16385), "channels"), (dict(dtype=F64, pdtype=F64, C=8193), "channels"),
                                         (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"), (dict(dtype=9), "dtype"),
                                         (dict(dtype=F16, pdtype=BF16), "weight dtype"), (dict(pdtype=F16), "weight dtype"), (dict(eps=-1.0), "eps"),
                                         (dict(eps=math.nan), "eps"), (dict(eps=math.inf), "eps"), (dict(x=None), "null"), (dict(y=None), "null"),
                                         (dict(sum="p"), "residual")])
def test_norm_refuses(change, text):
    p = _p()
    a = dict(x=p, res=None, w=p, sum=None, y=p, rows=2, C=8, eps=1e-6, dtype=F32, pdtype=F32)
    a.update({k: p if v == "p" else v for k, v in change.items()})
    rc = lib.gnnhwc_rms_fwd(a["x"], a["res"], a["w"], a["sum"], a["y"], a["rows"], a["C"], a["C"], a["C"], a["eps"], a["dtype"], a["pdtype"], None)
    assert rc == -1 and text in _cabi.last_error(), _cabi.last_error()


def test_quantised_norm_and_backward_refuse():
    p = _p()
    for block, dtype, qtype, text in ((100, F32, 4, "block"), (8, F32, 4, "block"), (512, F32, 4, "block"), (0, F64, 4, "8-bit"), (0, F32, 3, "8-bit type")):
        rc = lib.gnnhwc_rms_fwd_quant(p, None, None, None, p, p, 2, 1000, 1000, 0, block, 1e-6, dtype, dtype, qtype, None)
        assert rc == -1 and text in _cabi.last_error()
    assert lib.gnnhwc_rms_fwd_quant(p, None, None, None, p, None, 2, 8, 8, 0, 0, 1e-6, F32, F32, 4, None) == -1
    assert lib.gnnhwc_rms_bwd(None, None, p, p, p, p, 2, 8, 8, 8, 8, 1e-6, F32, F32, p, 1 << 20, None) == -1
    assert lib.gnnhwc_rms_bwd(p, None, p, p, p, p, 2, 8, 8, 8, 8, 1e-6, F32, F32, p, 16, None) == -2 and "workspace" in _cabi.last_error()
    assert lib.gnnhwc_rms_bwd(p, None, p, p, p, p, 2, 8, 8, 8, 8, 1e-6, F32, F32, None, 1 << 20, None) == -2
    # nothing asked for, or no rows: nothing to launch
    assert lib.gnnhwc_rms_bwd(p, None, p, p, None, None, 2, 8, 8, 8, 8, 1e-6, F32, F32, None, 0, None) == 0
    assert lib.gnnhwc_rms_fwd(None, None, None, None, None, 0, 8, 8, 8, 1e-6, F32, F32, None) == 0


def test_workspaces():
    assert lib.gnnhwc_rms_bwd_workspace_bytes(4, 20000, F32) == 0 and "channels" in _cabi.last_error()
    small, large = (lib.gnnhwc_rms_bwd_workspace_bytes(r, 1280, BF16) for r in (8, 1 << 20))
    assert 0 < small < large <= 16 << 20
    assert lib.gnnhwc_clip_workspace_bytes(0) > 0 and lib.gnnhwc_clip_workspace_bytes(5000) < 1 << 16
    assert lib.gnnhwc_clip_workspace_bytes(-1) == 0


def _call(**change):
    c = _cabi.RotaryCall()
    p = _p()
    c.q = c.k = c.q_grad = c.k_grad = c.q_out = c.k_out = c.positions = c.frequencies = p.value
    c.batch, c.tokens, c.heads, c.kv_heads, c.head_dim, c.axes, c.dtype, c.param_dtype, c.eps = 1, 2, 2, 1, 64, 2, BF16, BF16, 1e-6
    c.section_end[0], c.section_end[1] = 16, 32
    for k, v in change.items():
        if k == "ends":
            for i, e in enumerate(v):
                c.section_end[i] = e
        else:
            setattr(c, k, p.value if v == "p" else v)
    return c, p


@pytest.mark.parametrize("change,text", [(dict(head_dim=63), "even"), (dict(head_dim=0), "even"), (dict(head_dim=258), "256"), (dict(axes=0), "axes"),
                                         (dict(axes=5), "axes"), (dict(ends=(16, 8)), "descend"), (dict(ends=(16, 33)), "pairs"), (dict(ends=(0, 0)), "pairs"),
                                         (dict(position_type=3), "position_type"), (dict(heads=0), "heads"), (dict(heads=70000, kv_heads=0, k_out=None), "heads"),
                                         (dict(kv_heads=0), "kv_heads"), (dict(k_out=None), "kv_heads"), (dict(dtype=7), "dtype"),
                                         (dict(q_weight="p"), "together"), (dict(positions=None), "null"), (dict(frequencies=None), "null"),
                                         (dict(q=None), "null"), (dict(k=None), "null"), (dict(batch=2 ** 31, tokens=4), "tokens"), (dict(batch=2 ** 40, tokens=2 ** 40), "tokens"),
                                         (dict(batch=-1), "batch"), (dict(q_weight="p", k_weight="p", eps=-1.0), "eps"),
                                         (dict(q_weight="p", k_weight="p", param_dtype=F16), "weight dtype"),
                                         (dict(head_dim=254, ends=(8, 16)), "multiple of 8")])
def test_rotary_refuses(change, text):
    c, _keep = _call(**change)
    assert lib.gnnhwc_rotary(ctypes.byref(c), None) == -1 and text in _cabi.last_error(), _cabi.last_error()


def test_rotary_backward_refuses():
    c, _keep = _call(q_grad=None)
    assert lib.gnnhwc_rotary_bwd(ctypes.byref(c), None, 0, None) == -1 and "gradient" in _cabi.last_error()
    c, _keep = _call(q_weight="p", k_weight="p")
    assert lib.gnnhwc_rotary_bwd_workspace_bytes(ctypes.byref(c)) > 256
    assert lib.gnnhwc_rotary_bwd(ctypes.byref(c), None, 0, None) == -2
    assert lib.gnnhwc_rotary(None, None) == -1 and lib.gnnhwc_rotary_bwd(None, None, 0, None) == -1
    c, _keep = _call(tokens=0)
    assert lib.gnnhwc_rotary(ctypes.byref(c), None) == 0


def _clip(sizes, addresses, outs=None, types=None, **change):
    n = len(sizes)
    a = dict(max_norm=1.0, eps=1e-6, scale=1.0, total=_p(), total_dtype=F32, ws=_p(), nbytes=1 << 20, count=n)
    a.update(change)
    arr = lambda v: None if v is None else (ctypes.c_void_p * n)(*v)  # noqa: E731
    t = (ctypes.c_int * n)(*(types or [F32] * n))
    return lib.gnnhwc_clip(arr(addresses), arr(outs), (ctypes.c_int64 * n)(*sizes), t, t if outs is not None else None, a["count"], a["max_norm"], a["eps"],
                           a["scale"], a["total"], a["total_dtype"], a["ws"], a["nbytes"], None)


def test_clip_refuses():
    base = 1 << 30
    for kwargs, text in ((dict(max_norm=-1.0), "max_norm"), (dict(max_norm=math.nan), "max_norm"), (dict(eps=-1.0), "eps"), (dict(scale=math.inf), "grad_scale"),
                         (dict(scale=math.nan), "grad_scale"), (dict(total=None), "total"), (dict(total_dtype=F16), "total"), (dict(types=[F32, 8]), "dtype"),
                         (dict(count=-1), "count")):
        assert _clip([4, 4], [base, base + 64], **kwargs) == -1 and text in _cabi.last_error(), _cabi.last_error()
    assert _clip([4, 4], [base, base + 64], ws=None) == -2 and _clip([4, 4], [base, base + 64], nbytes=64) == -2
    # overlaps of what is written
    assert _clip([4, 4], [base, base + 12]) == -1 and "overlaps" in _cabi.last_error()
    assert _clip([100, 4], [base, base + 8]) == -1 and "overlaps" in _cabi.last_error()
    assert _clip([4, 4], [base, base + 64], [base + 64, base + 128]) == -1 and "overlaps" in _cabi.last_error()
    assert _clip([4, 4], [base, base + 64], [base + 128, base + 132]) == -1 and "overlaps" in _cabi.last_error()
    assert _clip([-1], [base]) == -1 and _clip([4], [None]) == -1


def test_python_surface():
    f = rotary_frequencies((4, 8), theta=100.0)
    assert f.dtype == torch.float32 and f.shape == (12,)
    assert torch.allclose(f[4:], 100.0 ** (-torch.arange(8) / 8)) and torch.allclose(rotary_frequencies((4, 8), 100.0, "head"), 100.0 ** (-torch.arange(12) / 12))
    with pytest.raises(ValueError):
        rotary_frequencies((4,), ladder="none")
    m = RMSNorm(16, channel_dim=1)
    assert isinstance(m, torch.nn.RMSNorm) and sorted(m.state_dict()) == ["weight"] and "channel_dim=1" in repr(m)
    m.load_state_dict(torch.nn.RMSNorm(16).state_dict())
    r = Rotary(64, (8, 12, 12), qk_norm=True)
    assert sorted(r.state_dict()) == ["k_weight", "q_weight"] and sorted(Rotary(64, (32,)).state_dict()) == []
    assert r.double().frequencies.dtype == torch.float32
    assert float(gnnhwc.clip_gradients([], 1.0)) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8)
    q = torch.zeros(1, 2, 1, 8)
    for call in (lambda: rms_norm(x), lambda: rms_norm(x, residual=x, return_sum=True), lambda: rms_norm_quant(x), lambda: RMSNorm(8)(x),
                 lambda: rotary(q, None, torch.zeros(2, 1), torch.ones(4)), lambda: gnnhwc.clip_gradients([x], 1.0)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()


def test_meta_kernels():
    x, w = torch.zeros((3, 5, 64), device="meta", dtype=torch.bfloat16), torch.zeros(64, device="meta")
    y, s = torch.ops.gnop.rms_norm(x, x, w, 1e-6, True)
    assert y.shape == s.shape == x.shape and y.dtype == x.dtype and torch.ops.gnop.rms_norm(x, None, w, 1e-6, True)[1].numel() == 0
    dx, dw = torch.ops.gnop.rms_norm_bwd(x, None, x, w, 1e-6)
    assert dx.shape == x.shape and dw.shape == w.shape and dw.dtype == w.dtype
    q, scales, s = torch.ops.gnop.rms_norm_quant(x, None, w, 1e-6, 32, torch.float8_e4m3fn, False)
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (3, 5, 2) and s.numel() == 0
    q = torch.zeros((2, 3, 4, 64), device="meta")
    a, b = torch.ops.gnop.rotary(q, q[:, :, :1], w, w, [32], False, None, None, 1e-6)
    assert a.shape == q.shape and b.shape == (2, 3, 1, 64)
