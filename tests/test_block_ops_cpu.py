"""Rotary positions, norms around a block and windowed attention, as far as no GPU is needed: the descriptors' layout, what
the C calls and the Python functions refuse, calls over nothing, and the table of frequencies."""
import ctypes
import inspect
import math
import os
import shutil
import subprocess
import sys

import pytest
import torch

import llmt_b200 as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MB = 1 << 20  # addresses below are multiples of it: none is ever read


# ------------------------------------------------------------------------------------------------------------- layout

STRUCTS = {"head_view": (L.HeadView, ["data", "stride_batch", "stride_head"]),
           "rope_desc": (L.RopeDesc, ["rot_dim", "x", "y", "freqs", "positions", "offset", "dtype", "inverse", "scale"]),
           "norm_residual_desc": (L.NormResidualDesc, ["groups", "dtype_res", "eps", "x", "out", "ld_x", "w_post", "rstd_post", "dout", "dx", "ld_dout",
                                                       "dw_post", "beta", "workspace", "workspace_bytes"]),
           "attention_desc": (L.AttentionDesc, ["window", "sinks", "scale", "dtype", "q", "out", "lse", "lengths", "dout", "dv", "workspace",
                                                "workspace_bytes"])}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_descriptor_layouts_match_the_header(tmp_path):
    lines, want = [], []
    for name, (cls, fields) in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof(llmt_b200_{name}));')
        want.append(ctypes.sizeof(cls))
        for f in fields:
            lines.append(f'printf("%zu\\n", offsetof(llmt_b200_{name}, {f}));')
            want.append(getattr(cls, f).offset)
    c = tmp_path / "layout.c"
    c.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"llmt_b200.h\"\nint main(void) {\n" + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)])
    assert [int(x) for x in subprocess.check_output([str(exe)]).split()] == want


NATIVE = ["rope", "norm_residual_fwd", "norm_residual_bwd", "attention_window_fwd", "attention_window_bwd", "attention_window_decode"]


@pytest.mark.parametrize("name", NATIVE)
def test_native_functions_keep_their_python_face(name):
    f = getattr(L, name)
    python = inspect.unwrap(f)
    assert f is not python, "the native form is in place"
    assert inspect.signature(f) == inspect.signature(python)
    assert (f.__name__, f.__module__, f.__doc__) == (name, "llmt_b200", python.__doc__)
    with pytest.raises(TypeError):
        f(no_such_argument=1)


def test_an_extension_from_before_these_functions_is_no_obstacle():
    """Importing (which building does first) over an extension that does not know a function leaves that function in Python."""
    code = ("import sys, types\n"
            "def fast(f):\n"
            "    if f.__name__ in %r: raise ValueError(f)\n"
            "    return f\n"
            "sys.modules['llmt_b200._native'] = types.SimpleNamespace(setup=lambda *a: None, fast=fast, NAMES=())\n"
            "import llmt_b200 as L, inspect\n"
            "assert inspect.isfunction(L.rope) and inspect.isfunction(L.attention_window_decode)\n" % NATIVE)
    subprocess.check_call([sys.executable, "-c", code], cwd=ROOT)


# ------------------------------------------------------------------------------------------------- rotary frequencies

@pytest.mark.parametrize("rot,base,factor,low,high,trained", [
    (64, 10000.0, 1.0, 1.0, 32.0, 0.0), (128, 500000.0, 8.0, 1.0, 4.0, 8192.0), (2, 10000.0, 4.0, 1.0, 32.0, 4096.0),
    (96, 10000.0, 2.0, math.inf, math.inf, 0.0), (64, 10000.0, 4.0, 2.0, 2.0, 2048.0), (0, 10000.0, 1.0, 1.0, 32.0, 0.0)])
def test_rope_frequencies_are_the_formula(rot, base, factor, low, high, trained):
    got = L.rope_frequencies(rot, base, factor, low, high, trained, device="cpu")
    assert got.dtype == torch.float64 and got.shape == (rot // 2,)
    for i, g in enumerate(got.tolist()):
        f = base ** (-2 * i / rot)
        turns = trained * f / (2 * math.pi)
        keep = 1.0 if factor == 1.0 or turns >= high else 0.0 if turns <= low else (turns - low) / (high - low)
        # each operation is off by 2^-53, powers by a few of those
        assert abs(g - f * (keep + (1 - keep) / factor)) <= 2.0 ** -48 * f


@pytest.mark.parametrize("args", [(3,), (-2,), (8, 0.0), (8, -1.0), (8, math.nan), (8, 10000.0, 0.0), (8, 10000.0, 2.0, 4.0, 1.0, 10.0),
                                  (8, 10000.0, 2.0, 1.0, 4.0, -1.0), (8, 10000.0, 2.0, math.nan, 4.0, 1.0)])
def test_rope_frequencies_refuse(args):
    with pytest.raises(L.LlmtB200Error):
        L.rope_frequencies(*args, device="cpu")


# ------------------------------------------------------------------------------------------------------------ C calls

def view(at, *strides):
    return L.HeadView(at, *strides)


def rope_desc(**kw):
    d = L.RopeDesc()
    d.batch, d.tokens, d.heads, d.head_dim, d.rot_dim = 2, 8, 4, 64, 64
    d.x, d.y = view(1 * MB, 2048, 256, 64), view(2 * MB, 2048, 256, 64)
    d.freqs, d.dtype, d.scale = 3 * MB, L.BF16, 1.0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,status,needle", [
    (dict(rot_dim=66), L.ERR_INVALID, "bad shape"),
    (dict(rot_dim=63), L.ERR_INVALID, "bad shape"),
    (dict(rot_dim=-2), L.ERR_INVALID, "bad shape"),
    (dict(batch=-1), L.ERR_INVALID, "bad shape"),
    (dict(head_dim=0, rot_dim=0), L.ERR_INVALID, "bad shape"),
    (dict(dtype=9), L.ERR_UNSUPPORTED, "dtype code 9"),
    (dict(head_dim=1032), L.ERR_UNSUPPORTED, "head_dim above 1024"),
    (dict(heads=65537), L.ERR_UNSUPPORTED, "heads above 65536"),
    (dict(batch=1 << 31), L.ERR_UNSUPPORTED, "blocks"),
    (dict(batch=1 << 20, tokens=1 << 20), L.ERR_UNSUPPORTED, "blocks"),
    (dict(freqs=None), L.ERR_INVALID, "null data"),
    (dict(x=view(None, 2048, 256, 64)), L.ERR_INVALID, "null data"),
    (dict(freqs=3 * MB + 4), L.ERR_INVALID, "aligned"),
    (dict(positions=4 * MB + 2), L.ERR_INVALID, "aligned"),
    (dict(y=view(2 * MB + 1, 2048, 256, 64)), L.ERR_INVALID, "aligned"),
    (dict(x=view(1 * MB, 2048, -256, 64)), L.ERR_INVALID, "strides"),
    (dict(x=view(1 * MB, 1 << 60, 256, 64)), L.ERR_INVALID, "strides"),
    (dict(y=view(2 * MB, 2048, 256, 32)), L.ERR_INVALID, "overlap one another"),
    (dict(y=view(2 * MB, 0, 256, 64)), L.ERR_INVALID, "overlap one another"),
    (dict(y=view(1 * MB + 128, 2048, 256, 64)), L.ERR_INVALID, "y must be x"),
    (dict(y=view(1 * MB, 2048, 64, 512)), L.ERR_INVALID, "y must be x"),
    (dict(freqs=2 * MB + 64), L.ERR_INVALID, "freqs or positions"),
    (dict(positions=2 * MB), L.ERR_INVALID, "freqs or positions"),
])
def test_rope_refuses(kw, status, needle):
    assert L.lib().llmt_b200_rope(ctypes.byref(rope_desc(**kw)), None) == status
    assert needle in L.last_error()


@pytest.mark.parametrize("kw", [dict(batch=0), dict(tokens=0), dict(heads=0), dict(rot_dim=0, y=view(1 * MB, 2048, 256, 64), freqs=None)])
def test_rope_of_nothing_is_done(kw):
    before = L.launch_count()
    assert L.lib().llmt_b200_rope(ctypes.byref(rope_desc(**kw)), None) == L.OK and L.launch_count() == before


def norm_desc(back=False, **kw):
    d = L.NormResidualDesc()
    d.rows, d.cols, d.groups, d.dtype_res, d.dtype_act, d.scale, d.eps = 16, 64, 2, L.FP32, L.BF16, 1.0, 1e-5
    for i, n in enumerate(["x", "y", "out", "h"] + (["dout", "dh", "dx", "dy"] if back else [])):
        setattr(d, n, (1 + i) * MB)
        setattr(d, "ld_" + n, 64)
    for i, n in enumerate(["w_post", "gate", "w_pre", "rstd_post", "rstd_pre"] + (["dw_post", "dgate", "dw_pre", "workspace"] if back else [])):
        setattr(d, n, (20 + i) * MB)
    d.workspace_bytes = MB
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BOTH = [
    (dict(cols=0), L.ERR_INVALID, "bad shape"),
    (dict(rows=-1), L.ERR_INVALID, "bad shape"),
    (dict(groups=3), L.ERR_INVALID, "bad shape"),
    (dict(groups=0), L.ERR_INVALID, "bad shape"),
    (dict(dtype_act=7), L.ERR_UNSUPPORTED, "dtype codes"),
    (dict(dtype_res=L.BF16, dtype_act=L.FP32), L.ERR_UNSUPPORTED, "dtype codes"),
    (dict(cols=16385), L.ERR_UNSUPPORTED, "columns"),
    (dict(rows=1 << 31), L.ERR_UNSUPPORTED, "rows"),
    (dict(y=None), L.ERR_INVALID, "belong to y"),
    (dict(w_post=20 * MB + 2), L.ERR_INVALID, "aligned"),
    (dict(y=2 * MB + 1), L.ERR_INVALID, "aligned"),
    (dict(ld_y=-64), L.ERR_INVALID, "row pitch of y"),
    (dict(ld_y=1 << 29), L.ERR_INVALID, "row pitch of y"),
]


@pytest.mark.parametrize("kw,status,needle", BOTH + [
    (dict(x=None), L.ERR_INVALID, "null data"),
    (dict(out=None), L.ERR_INVALID, "null data"),
    (dict(h=None), L.ERR_INVALID, "go together"),
    (dict(w_pre=None), L.ERR_INVALID, "go together"),
    (dict(y=None, w_post=None, gate=None, h=None, w_pre=None), L.ERR_INVALID, "nothing to do"),
    (dict(ld_out=32), L.ERR_INVALID, "row pitch of out"),
    (dict(out=2 * MB + 64), L.ERR_INVALID, "out overlaps y"),
    (dict(out=1 * MB + 4), L.ERR_INVALID, "out overlaps x"),
    (dict(out=1 * MB, ld_out=128), L.ERR_INVALID, "out overlaps x"),
    (dict(h=3 * MB), L.ERR_INVALID, "out overlaps h"),
    (dict(w_pre=3 * MB), L.ERR_INVALID, "w_pre overlaps out"),
    (dict(rstd_pre=4 * MB), L.ERR_INVALID, "rstd_pre overlaps h"),
    (dict(rstd_post=24 * MB), L.ERR_INVALID, "rstd_post overlaps rstd_pre"),
])
def test_norm_residual_fwd_refuses(kw, status, needle):
    assert L.lib().llmt_b200_norm_residual_fwd(ctypes.byref(norm_desc(**kw)), None) == status
    assert needle in L.last_error()


@pytest.mark.parametrize("kw,status,needle", BOTH + [
    (dict(dx=None), L.ERR_INVALID, "null data"),
    (dict(dout=None, dh=None, w_pre=None, dw_pre=None), L.ERR_INVALID, "null data"),
    (dict(out=None), L.ERR_INVALID, "null data"),
    (dict(rstd_pre=None), L.ERR_INVALID, "null data"),
    (dict(rstd_post=None), L.ERR_INVALID, "null data"),
    (dict(dy=None), L.ERR_INVALID, "null data"),
    (dict(dh=None), L.ERR_INVALID, "go together"),
    (dict(w_post=None), L.ERR_INVALID, "null"),
    (dict(gate=None), L.ERR_INVALID, "null"),
    (dict(dw_pre=27 * MB + 1), L.ERR_INVALID, "aligned"),
    (dict(ld_dx=32), L.ERR_INVALID, "row pitch of dx"),
    (dict(dx=3 * MB), L.ERR_INVALID, "dx overlaps out"),
    (dict(dy=2 * MB), L.ERR_INVALID, "dy overlaps y"),
    (dict(dx=5 * MB, ld_dx=128), L.ERR_INVALID, "overlaps"),
    (dict(dw_post=20 * MB), L.ERR_INVALID, "dw_post overlaps w_post"),
    (dict(dgate=25 * MB), L.ERR_INVALID, "overlaps"),
    (dict(dw_pre=7 * MB), L.ERR_INVALID, "dw_pre overlaps dx"),
    (dict(w_pre=8 * MB), L.ERR_INVALID, "w_pre overlaps dy"),
    (dict(workspace=None), L.ERR_WORKSPACE, "bytes needed"),
    (dict(workspace_bytes=16), L.ERR_WORKSPACE, "bytes needed"),
    (dict(workspace=28 * MB + 8), L.ERR_INVALID, "16-byte aligned"),
    (dict(workspace=7 * MB), L.ERR_INVALID, "workspace overlaps dx"),
    (dict(workspace=22 * MB), L.ERR_INVALID, "workspace overlaps w_pre"),
])
def test_norm_residual_bwd_refuses(kw, status, needle):
    assert L.lib().llmt_b200_norm_residual_bwd(ctypes.byref(norm_desc(True, **kw)), None) == status
    assert needle in L.last_error()


def test_norm_residual_of_no_rows_is_done():
    before = L.launch_count()
    assert L.lib().llmt_b200_norm_residual_fwd(ctypes.byref(norm_desc(rows=0)), None) == L.OK
    assert L.lib().llmt_b200_norm_residual_bwd(ctypes.byref(norm_desc(True, rows=0, beta=1.0)), None) == L.OK
    assert L.launch_count() == before
    assert L.lib().llmt_b200_norm_residual_bwd(ctypes.byref(norm_desc(True, rows=0, beta=0.5)), None) == L.ERR_UNSUPPORTED


def attn_desc(back=False, **kw):
    """2 sequences, 4 heads on 2, 16 queries on 32 keys of 64; each tensor in a megabyte of its own."""
    d = L.AttentionDesc()
    d.batch, d.heads, d.kv_heads, d.tokens_q, d.tokens_k, d.head_dim, d.scale, d.dtype = 2, 4, 2, 16, 32, 64, 0.125, L.BF16
    for i, n in enumerate(["q", "out"] + (["dout", "dq"] if back else [])):
        setattr(d, n, view((1 + i) * MB, 16 * 256, 256, 64))
    for i, n in enumerate(["k", "v"] + (["dk", "dv"] if back else [])):
        setattr(d, n, view((10 + i) * MB, 32 * 128, 128, 64))
    d.lse, d.workspace, d.workspace_bytes = 20 * MB, 21 * MB, 8 * MB
    for k, v in kw.items():
        setattr(d, k, v)
    return d


SHAPES = [
    (dict(batch=-1), L.ERR_INVALID, "negative"),
    (dict(sinks=-1), L.ERR_INVALID, "negative"),
    (dict(head_dim=0), L.ERR_INVALID, "negative"),
    (dict(kv_heads=3), L.ERR_INVALID, "multiple of kv_heads"),
    (dict(kv_heads=0), L.ERR_INVALID, "multiple of kv_heads"),
    (dict(dtype=L.FP32), L.ERR_UNSUPPORTED, "bf16 only"),
    (dict(head_dim=136), L.ERR_UNSUPPORTED, "multiple of 8 up to 128"),
    (dict(head_dim=60), L.ERR_UNSUPPORTED, "multiple of 8 up to 128"),
    (dict(tokens_k=1 << 31), L.ERR_UNSUPPORTED, "2^31"),
    (dict(batch=1 << 20, tokens_k=1 << 20), L.ERR_UNSUPPORTED, "rows over all heads"),
    (dict(scale=0.0), L.ERR_INVALID, "scale"),
    (dict(scale=-1.0), L.ERR_INVALID, "scale"),
    (dict(scale=math.nan), L.ERR_INVALID, "scale"),
    (dict(scale=math.inf), L.ERR_INVALID, "scale"),
    (dict(lse=20 * MB + 2), L.ERR_INVALID, "aligned"),
    (dict(k=view(None, 32 * 128, 128, 64)), L.ERR_INVALID, "tensor k"),
    (dict(k=view(10 * MB, 0, 128, 64)), L.ERR_INVALID, "k is broadcast"),
    (dict(v=view(11 * MB, 32 * 128, 128, 0)), L.ERR_INVALID, "v is broadcast"),
    (dict(q=view(1 * MB + 2, 16 * 256, 256, 64)), L.ERR_INVALID, "q needs"),
    (dict(v=view(11 * MB, 32 * 128, 132, 64)), L.ERR_INVALID, "v needs"),
    (dict(k=view(10 * MB, -32 * 128, 128, 64)), L.ERR_INVALID, "strides of k"),
    (dict(out=view(1 * MB, 16 * 256, 256, 64)), L.ERR_INVALID, "out overlaps q"),
]


@pytest.mark.parametrize("kw,status,needle", SHAPES + [
    (dict(out=view(2 * MB, 16 * 256, 256, 32)), L.ERR_INVALID, "overlap one another"),
    (dict(out=view(2 * MB, 256, 256, 64)), L.ERR_INVALID, "overlap one another"),
    (dict(out=view(11 * MB + 4096, 16 * 256, 256, 64)), L.ERR_INVALID, "out overlaps v"),
    (dict(lse=2 * MB), L.ERR_INVALID, "lse overlaps out"),
    (dict(lse=10 * MB + 64), L.ERR_INVALID, "lse overlaps k"),
    (dict(lengths=30 * MB), L.ERR_INVALID, "lengths belong"),
])
def test_attention_window_fwd_refuses(kw, status, needle):
    assert L.lib().llmt_b200_attention_window_fwd(ctypes.byref(attn_desc(**kw)), None) == status
    assert needle in L.last_error()


def test_attention_window_fwd_refuses_a_workspace_on_a_tensor():
    """64 queries on 8192 keys: done in parts, whose workspace is checked like any other (one that is too small is not used)."""
    d = dict(batch=1, tokens_q=64, tokens_k=8192, q=view(1 * MB, 0, 256, 64), out=view(2 * MB, 0, 256, 64), k=view(100 * MB, 0, 128, 64), v=view(110 * MB, 0, 128, 64),
             workspace_bytes=80 * MB)
    lib = L.lib()
    assert 0 < lib.llmt_b200_attention_window_fwd_workspace_bytes(ctypes.byref(attn_desc(**d))) <= 60 * MB
    for at, needle in ((21 * MB + 8, "16-byte aligned"), (100 * MB, "workspace overlaps k"), (2 * MB + 64, "workspace overlaps out"), (20 * MB, "workspace overlaps lse")):
        assert lib.llmt_b200_attention_window_fwd(ctypes.byref(attn_desc(**d, workspace=at)), None) == L.ERR_INVALID and needle in L.last_error()


@pytest.mark.parametrize("kw,status,needle", [s for s in SHAPES if "out" not in s[0]] + [
    (dict(dout=view(3 * MB, 16 * 256, 256, 0)), L.ERR_INVALID, "dout is broadcast"),
    (dict(dq=view(1 * MB, 16 * 256, 256, 64)), L.ERR_INVALID, "dq overlaps q"),
    (dict(dk=view(13 * MB, 32 * 128, 128, 64)), L.ERR_INVALID, "dk overlaps dv"),
    (dict(dv=view(13 * MB, 32 * 128, 64, 64)), L.ERR_INVALID, "overlap one another"),
    (dict(lse=None), L.ERR_INVALID, "lse"),
    (dict(lse=4 * MB), L.ERR_INVALID, "lse overlaps dq"),
    (dict(workspace=None), L.ERR_WORKSPACE, "bytes needed"),
    (dict(workspace_bytes=64), L.ERR_WORKSPACE, "bytes needed"),
    (dict(workspace=21 * MB + 4), L.ERR_INVALID, "16-byte aligned"),
    (dict(workspace=3 * MB + 64), L.ERR_INVALID, "workspace overlaps dout"),
    (dict(workspace=20 * MB), L.ERR_INVALID, "workspace overlaps lse"),
    (dict(lengths=30 * MB), L.ERR_INVALID, "lengths belong"),
])
def test_attention_window_bwd_refuses(kw, status, needle):
    assert L.lib().llmt_b200_attention_window_bwd(ctypes.byref(attn_desc(True, **kw)), None) == status
    assert needle in L.last_error()


def decode_desc(**kw):
    """2 sequences, 4 heads on 2, a cache of 65536 places of 64 (chunks: a workspace is needed)."""
    d = attn_desc(tokens_q=1, tokens_k=65536, lengths=40 * MB)
    d.q, d.out = view(1 * MB, 256, 0, 64), view(2 * MB, 256, 0, 64)
    d.k, d.v = view(100 * MB, 65536 * 128, 128, 64), view(200 * MB, 65536 * 128, 128, 64)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw,status,needle", [
    (dict(tokens_q=2), L.ERR_INVALID, "tokens_q must be 1"),
    (dict(tokens_q=0), L.ERR_INVALID, "tokens_q must be 1"),
    (dict(lengths=40 * MB + 2), L.ERR_INVALID, "aligned"),
    (dict(lengths=2 * MB), L.ERR_INVALID, "lengths overlaps out"),
    (dict(lengths=20 * MB), L.ERR_INVALID, "lse overlaps lengths"),
    (dict(out=view(1 * MB, 256, 0, 64)), L.ERR_INVALID, "out overlaps q"),
    (dict(v=view(200 * MB, 65536 * 128, 0, 64)), L.ERR_INVALID, "v is broadcast"),
    (dict(workspace=None), L.ERR_WORKSPACE, "bytes needed"),
    (dict(workspace=21 * MB + 8), L.ERR_INVALID, "16-byte aligned"),
    (dict(workspace=100 * MB), L.ERR_INVALID, "workspace overlaps k"),
    (dict(workspace=40 * MB), L.ERR_INVALID, "workspace overlaps lse or lengths"),
])
def test_attention_window_decode_refuses(kw, status, needle):
    assert L.lib().llmt_b200_attention_window_decode(ctypes.byref(decode_desc(**kw)), None) == status
    assert needle in L.last_error()


@pytest.mark.parametrize("kw", [dict(batch=0), dict(heads=0, kv_heads=0), dict(tokens_q=0, tokens_k=0)])
def test_attention_of_nothing_is_done(kw):
    before = L.launch_count()
    assert L.lib().llmt_b200_attention_window_fwd(ctypes.byref(attn_desc(**kw)), None) == L.OK
    assert L.lib().llmt_b200_attention_window_bwd(ctypes.byref(attn_desc(True, **kw)), None) == L.OK
    if "tokens_q" not in kw:
        assert L.lib().llmt_b200_attention_window_decode(ctypes.byref(decode_desc(**kw)), None) == L.OK
    assert L.launch_count() == before


@pytest.mark.parametrize("name", ["rope", "norm_residual_fwd", "norm_residual_bwd", "attention_window_fwd", "attention_window_bwd", "attention_window_decode"])
def test_a_null_descriptor_is_refused(name):
    assert getattr(L.lib(), "llmt_b200_" + name)(None, None) == L.ERR_INVALID and "null descriptor" in L.last_error()


def test_workspace_queries_answer_nothing_for_bad_descriptors():
    lib = L.lib()
    assert lib.llmt_b200_norm_residual_workspace_bytes(ctypes.byref(norm_desc(True, cols=0))) == 0
    assert lib.llmt_b200_attention_window_workspace_bytes(ctypes.byref(attn_desc(True, kv_heads=3))) == 0
    assert lib.llmt_b200_attention_window_decode_workspace_bytes(ctypes.byref(decode_desc(head_dim=12))) == 0
    assert lib.llmt_b200_attention_window_fwd_workspace_bytes(ctypes.byref(attn_desc(head_dim=4))) == 0
    for f in ("norm_residual_workspace_bytes", "attention_window_workspace_bytes", "attention_window_fwd_workspace_bytes", "attention_window_decode_workspace_bytes"):
        assert getattr(lib, "llmt_b200_" + f)(None) == 0


# --------------------------------------------------------------------------------------------------- Python functions

def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


python = inspect.unwrap


def refused(call, needle):
    with pytest.raises(L.LlmtB200Error) as e:
        call()
    assert needle in str(e.value)


def test_python_refuses_tensors_that_are_not_on_a_gpu():
    f32 = torch.float32
    x, w, s = t(4, 64), t(64, dtype=f32), t(4, dtype=f32)
    q, k = t(1, 4, 2, 64), t(1, 4, 1, 64)
    refused(lambda: L.rope(t(1, 4, 2, 64), q, t(32, dtype=torch.float64)), "CUDA device")
    refused(lambda: L.norm_residual_fwd(t(4, 64), t(4, 64), x, t(4, 64), w_pre=w), "CUDA device")
    refused(lambda: L.norm_residual_bwd(t(4, 64), None, t(4, 64), t(4, 64), x, w_pre=w, rstd_pre=s), "CUDA device")
    refused(lambda: L.attention_window_fwd(t(1, 4, 2, 64), None, q, k, t(1, 4, 1, 64)), "CUDA device")
    refused(lambda: L.attention_window_bwd(t(1, 4, 2, 64), t(1, 4, 1, 64), t(1, 4, 1, 64), t(1, 4, 2, 64), q, k, t(1, 4, 1, 64), t(1, 4, 2, 64),
                                           t(1, 2, 4, dtype=f32)), "CUDA device")
    refused(lambda: L.attention_window_decode(t(1, 2, 64), t(1, 2, 64), k, t(1, 4, 1, 64)), "CUDA device")


def test_python_refuses_shapes_and_types():
    f64, f32 = torch.float64, torch.float32
    x, fr = t(2, 4, 2, 64), t(32, dtype=f64)
    refused(lambda: L.rope(t(2, 4, 2, 32), x, fr), "one shape and type")
    refused(lambda: L.rope(t(2, 4, 2, 64, dtype=f32), x, fr), "one shape and type")
    refused(lambda: L.rope(t(4, 2, 64), x, fr), "contiguous head_dim")
    refused(lambda: L.rope(x, t(2, 4, 64, 2).transpose(2, 3), fr), "contiguous head_dim")
    refused(lambda: L.rope(x, x, t(32, dtype=f32)), "freqs")
    refused(lambda: L.rope(x, x, t(64, dtype=f64)[::2]), "freqs")
    refused(lambda: L.rope(x, x, fr, positions=torch.zeros(2, 4, dtype=torch.int64)), "positions")
    refused(lambda: L.rope(x, x, fr, positions=torch.zeros(2, 3, dtype=torch.int32)), "positions")
    refused(lambda: L.rope(x, x, fr, positions=torch.zeros(4, 2, dtype=torch.int32).t()), "positions")
    r, w = t(4, 64), t(64, dtype=f32)
    refused(lambda: L.norm_residual_fwd(t(4, 32), None, r, t(4, 64)), "shape")
    refused(lambda: L.norm_residual_fwd(t(4, 64), None, r, t(64, 4).t()), "contiguous rows")
    refused(lambda: L.norm_residual_fwd(t(4, 64, dtype=f32), None, r, t(4, 64)), "another type")
    refused(lambda: L.norm_residual_fwd(t(4, 64, dtype=torch.float16), None, t(4, 64, dtype=torch.float16), t(4, 64)), "fp32 or bf16")
    refused(lambda: L.norm_residual_fwd(t(4, 64), t(4, 64), r, t(4, 64), w_pre=t(32, dtype=f32)), "w_pre")
    refused(lambda: L.norm_residual_fwd(t(4, 64), t(4, 64), r, t(4, 64), w_pre=t(64)), "w_pre")
    refused(lambda: L.norm_residual_fwd(t(4, 64), None, r, t(4, 64), gate=t(2, 32, dtype=f32)), "gate")
    refused(lambda: L.norm_residual_fwd(t(2, 2, 64), None, t(2, 4, 64)[:, ::2], t(2, 4, 64)[:, 1:3]), "evenly spaced")
    refused(lambda: L.norm_residual_bwd(t(4, 64), t(4, 64), t(4, 64), None, None, t(4, 64), gate=t(1, 64, dtype=f32), dgate=t(2, 64, dtype=f32)), "dgate")
    q, k = t(2, 4, 4, 64), t(2, 4, 2, 64)
    refused(lambda: L.attention_window_fwd(q, None, q, k, t(2, 4, 4, 64)), "k and v must be")
    refused(lambda: L.attention_window_fwd(q, None, q, k[:1], k[:1]), "k and v must be")
    refused(lambda: L.attention_window_fwd(t(2, 4, 4, 32), None, q, k, k), "out must have")
    refused(lambda: L.attention_window_fwd(t(2, 4, 4, 64, dtype=f32), None, q, k, k), "another type")
    refused(lambda: L.attention_window_fwd(q, t(2, 4, 4), q, k, k), "lse")
    refused(lambda: L.attention_window_fwd(q, t(2, 4, 3, dtype=f32), q, k, k), "lse")
    refused(lambda: L.attention_window_decode(t(2, 4, 64), q, k, k), "[batch, heads, head_dim]")
    refused(lambda: L.attention_window_decode(t(2, 4, 64), t(2, 4, 64), k, k, lengths=torch.zeros(2, dtype=torch.int64)), "lengths")
    refused(lambda: L.attention_window_decode(t(2, 4, 64), t(2, 4, 64), k, k, lengths=torch.zeros(3, dtype=torch.int32)), "lengths")
    flat = torch.zeros(1, dtype=torch.uint8).expand(1 << 20)   # a megabyte in name only
    gpu = lambda: pytest.MonkeyPatch.context()
    with gpu() as m:
        m.setattr(L, "_device_of", lambda *a: None)
        m.setattr(L, "_on", lambda device, stream, call: call(None))
        wf = t(64, dtype=f32)
        for call in (lambda: python(L.attention_window_fwd)(q, None, q, k, k, workspace=flat),
                     lambda: python(L.attention_window_bwd)(q, k, k, q, q, k, k, q, t(2, 4, 4, dtype=f32), workspace=flat),
                     lambda: python(L.attention_window_decode)(t(2, 4, 64), t(2, 4, 64), k, k, workspace=flat),
                     lambda: python(L.norm_residual_bwd)(t(4, 64), None, None, t(4, 64), t(4, 64), w_pre=wf, rstd_pre=t(4, dtype=f32), dw_pre=wf, workspace=flat)):
            refused(call, "workspace must be contiguous")
