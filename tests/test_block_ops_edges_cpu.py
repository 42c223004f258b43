"""Rotary positions, norms around a block and windowed attention: calls at the edge of what the header allows, as far as no GPU
is needed (an accepted call ends at the missing workspace or at the launch)."""
import ctypes
import inspect
import itertools
import os
import random
import re
import subprocess
import sys

import pytest
import torch

import llmt_b200 as L
from tests.test_block_ops_cpu import MB, ROOT, attn_desc, decode_desc, norm_desc, rope_desc, view

BF = dict(dtype_res=L.BF16, dtype_act=L.BF16)


@pytest.mark.parametrize("kw,needle", [
    (dict(out=1 * MB, h=1 * MB), "overlaps h"),   # out may be x, h is a result of its own
    (dict(out=1 * MB, y=1 * MB), "out overlaps y"),
    (dict(out=1 * MB, ld_out=128), "out overlaps x"),
])
def test_norm_residual_fwd_in_place_shares_nothing_else(kw, needle):
    assert L.lib().llmt_b200_norm_residual_fwd(ctypes.byref(norm_desc(**BF, **kw)), None) == L.ERR_INVALID
    assert needle in L.last_error()


@pytest.mark.parametrize("kw,needle", [
    (dict(dx=5 * MB, dy=5 * MB), "overlaps"),     # dx may be dout (at 5 MB), dy is a result of its own
    (dict(dx=5 * MB, dh=5 * MB), "dx overlaps dh"),
    (dict(dx=5 * MB, out=5 * MB), "dx overlaps out"),
])
def test_norm_residual_bwd_in_place_shares_nothing_else(kw, needle):
    assert L.lib().llmt_b200_norm_residual_bwd(ctypes.byref(norm_desc(True, **BF, **kw)), None) == L.ERR_INVALID
    assert needle in L.last_error()


def test_norm_residual_in_place_is_accepted():
    lib = L.lib()
    # one row has no pitch; the backward call ends at the workspace that it is not given
    for kw in (dict(dx=5 * MB), dict(dx=5 * MB, rows=1, groups=1, ld_dx=1024)):
        assert lib.llmt_b200_norm_residual_bwd(ctypes.byref(norm_desc(True, **BF, workspace=None, **kw)), None) == L.ERR_WORKSPACE


def test_attention_without_query_heads_has_key_gradients():
    """dk and dv have elements and are to be zeroed: the call goes on to its launch, which fails here."""
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real")
    before = L.launch_count()
    assert L.lib().llmt_b200_attention_window_bwd(ctypes.byref(attn_desc(True, heads=0, lse=None)), None) != L.OK and L.launch_count() > before
    for kw in (dict(heads=0, kv_heads=0), dict(heads=0, tokens_k=0), dict(heads=0, batch=0)):
        before = L.launch_count()
        assert L.lib().llmt_b200_attention_window_bwd(ctypes.byref(attn_desc(True, lse=None, **kw)), None) == L.OK and L.launch_count() == before


def test_an_extension_of_other_sources_leaves_every_function_in_python():
    """One that lacks the block's functions: the functions that it has are not taken from it either, since it binds other
    arguments.  (The call is over nothing, and reaches torch's stream at most.)"""
    code = ("import sys, types, inspect\n"
            "def setup(binder, *rest): fake.binder = binder\n"
            "def bind(entries, raw_stream, get_device, float32, bfloat16, int32, desc): pass\n"
            "def fast(f):\n"
            "    if f.__name__ not in fake.NAMES: raise ValueError(f)\n"
            "    def call(*a, **k): fake.binder()\n"
            "    return call\n"
            "fake = types.SimpleNamespace(setup=setup, bind=bind, fast=fast, NAMES=('gemm', 'softmax_fwd', 'rowdot'))\n"
            "sys.modules['llmt_b200._native'] = fake\n"
            "import torch, llmt_b200 as L\n"
            "assert all(inspect.isfunction(getattr(L, n)) and getattr(L, n).__name__ == n for n in ('gemm', 'softmax_fwd', 'rowdot', 'rope'))\n"
            "try: L.gemm(torch.empty(0, 8), torch.empty(0, 4), torch.empty(4, 8))\n"
            "except TypeError: raise\n"
            "except Exception: pass\n")
    subprocess.check_call([sys.executable, "-c", code], cwd=ROOT)


def test_the_extension_of_these_sources_is_in_place():
    from llmt_b200 import _native
    assert tuple(_native.NAMES) == L._NATIVE_ENTRIES and not inspect.isfunction(L.gemm)


def _bytes_of(base, shape, strides, hd, size):
    runs = [base + size * sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, shape))]
    return {r + k for r in runs for k in range(0, hd * size, size)}   # element by element: all are aligned to their size


def _nested(rng, extents, unit, pad):
    """Strides of dimensions in a random order of nesting, each with up to `pad` units between."""
    order, strides, at = rng.sample(range(3), 3), [0, 0, 0], unit
    for i in order:
        strides[i] = at
        at = at * extents[i] + unit * rng.choice((0, 0, 1, pad))
    return strides, at


def test_gradients_may_lie_between_each_others_rows():
    """dq, dk and dv as views of one buffer are refused where they share an element, and only there.  (An accepted call ends at
    the workspace that it is not given.)"""
    rng, lib, base, seen = random.Random(5), L.lib(), 50 * MB, {True: 0, False: 0}
    for _ in range(1500):
        b, hkv, hd = rng.randint(1, 3), rng.randint(1, 2), 8
        h, tq, tk = hkv * rng.randint(1, 2), rng.randint(1, 4), rng.randint(1, 4)
        shapes = dict(dq=(b, tq, h), dk=(b, tk, hkv), dv=(b, tk, hkv))
        common, span = _nested(rng, (b, max(tq, tk), h + 2 * hkv), hd, 3)
        at, parts = {}, {}
        for n, first in (("dq", 0), ("dk", h), ("dv", h + hkv)):
            if rng.random() < 0.7:   # of the common buffer, mostly in its own place there
                strides, off = common, common[2] * first if rng.random() < 0.8 else 8 * rng.randint(0, span // 8)
            else:
                strides, off = _nested(rng, shapes[n], hd, 3)[0], 8 * rng.randint(0, span // 8)
            at[n], parts[n] = view(base + 2 * off, *strides), _bytes_of(base + 2 * off, shapes[n], strides, hd, 2)
        meet = any(parts[x] & parts[y] for x, y in (("dq", "dk"), ("dq", "dv"), ("dk", "dv")))
        d = attn_desc(True, batch=b, heads=h, kv_heads=hkv, tokens_q=tq, tokens_k=tk, head_dim=hd, workspace=None, **at)
        status = lib.llmt_b200_attention_window_bwd(ctypes.byref(d), None)
        assert status == (L.ERR_INVALID if meet else L.ERR_WORKSPACE), (b, h, hkv, tq, tk, meet, L.last_error())
        assert not meet or "overlaps" in L.last_error()
        seen[meet] += 1
    assert min(seen.values()) > 200


@pytest.mark.parametrize("batch", [1, 2, 64])
@pytest.mark.parametrize("order", ["bhtd", "bthd", "hbtd", "thbd"])
def test_packed_gradients_of_any_order_are_accepted(batch, order):
    h, hkv, t, hd = 8, 2, 4096, 64
    n, at, strides = dict(b=batch, t=t, h=h + 2 * hkv), hd, {}
    for dim in reversed(order[:3]):
        strides[dim] = at
        at *= n[dim]
    where = lambda first: view(50 * MB + 2 * first * strides["h"], strides["b"], strides["t"], strides["h"])
    d = attn_desc(True, batch=batch, heads=h, kv_heads=hkv, tokens_q=t, tokens_k=t, workspace=None, dq=where(0), dk=where(h), dv=where(h + hkv))
    for i, name in enumerate(["q", "out", "dout", "k", "v"]):
        setattr(d, name, view((4096 + 1024 * i) * MB, t * h * hd, h * hd, hd))
    d.lse = 16384 * MB
    assert L.lib().llmt_b200_attention_window_bwd(ctypes.byref(d), None) == L.ERR_WORKSPACE, L.last_error()
    d.dv = where(h + hkv - 1)   # dk's last head
    assert L.lib().llmt_b200_attention_window_bwd(ctypes.byref(d), None) == L.ERR_INVALID and "dk overlaps dv" in L.last_error()


def test_rope_may_write_between_the_rows_that_it_reads():
    """x and y in one buffer are refused where they share an element, and only there (the frequencies lie on y, which ends the call
    before it begins)."""
    rng, lib, base, seen = random.Random(6), L.lib(), 50 * MB, {True: 0, False: 0}
    for _ in range(800):
        shape, hd = [rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 3)], rng.choice((2, 4, 6))
        (xs, span), (ys, _) = (_nested(rng, (shape[0], shape[1], 2 * shape[2]), hd, 3) for _ in range(2))
        off = rng.randint(0, span)
        if rng.random() < 0.5:   # y: the heads behind x's
            ys, off = xs, xs[2] * shape[2]
        if rng.random() < 0.2:
            xs = [0] + xs[1:]    # one sequence read for all
        x, y = _bytes_of(base, shape, xs, hd, 4), _bytes_of(base + 4 * off, shape, ys, hd, 4)
        same = off == 0 and all(n == 1 or a == b for n, a, b in zip(shape, xs, ys))
        d = rope_desc(batch=shape[0], tokens=shape[1], heads=shape[2], head_dim=hd, rot_dim=0 if same else 2, dtype=L.FP32, x=view(base, *xs),
                      y=view(base + 4 * off, *ys), freqs=base + 4 * off // 8 * 8)
        status = lib.llmt_b200_rope(ctypes.byref(d), None)
        if same:
            assert status == L.OK
            continue
        meet = bool(x & y)
        # where x and y are apart the frequencies are what is refused: they lie on y
        assert status == L.ERR_INVALID and ("y must be x" in L.last_error()) == meet, (shape, hd, xs, ys, off)
        assert meet or "freqs" in L.last_error()
        seen[meet] += 1
    assert min(seen.values()) > 100


def test_norm_residual_may_write_between_the_rows_that_it_reads():
    """dx among the rows of the other tensors is refused where they share an element, and only there."""
    rng, lib, base, seen = random.Random(7), L.lib(), 50 * MB, {True: 0, False: 0}
    for _ in range(600):
        rows, cols, pitch = rng.randint(1, 6), rng.randint(1, 5), rng.randint(5, 12)
        other, off = (pitch, rng.randint(0, 2 * pitch)) if rng.random() < 0.6 else (rng.randint(5, 12), rng.randint(0, 40))
        meet = bool(_bytes_of(base, (rows, 1, 1), (pitch, 0, 0), cols, 4) & _bytes_of(base + 4 * off, (rows, 1, 1), (other, 0, 0), cols, 4))
        name = rng.choice(["out", "dout"])
        if name == "dout" and off == 0 and (rows == 1 or pitch == other):
            continue   # in place
        kw = {"dx": base, "ld_dx": pitch, name: base + 4 * off, "ld_" + name: other}
        status = lib.llmt_b200_norm_residual_bwd(ctypes.byref(norm_desc(True, rows=rows, cols=cols, groups=1, workspace=None, **kw)), None)
        assert status == (L.ERR_INVALID if meet else L.ERR_WORKSPACE), (rows, cols, pitch, other, off, L.last_error())
        seen[meet] += 1
    assert min(seen.values()) > 100


@pytest.mark.parametrize("kw,status", [
    (dict(batch=128, heads=128, kv_heads=8, tokens_k=131072, head_dim=128), L.ERR_WORKSPACE),   # 2^31 rows, 69 GB of keys and values
    (dict(batch=1 << 20, heads=1, kv_heads=1, tokens_k=4096), L.ERR_WORKSPACE),
    (dict(batch=1 << 20, heads=2048, kv_heads=1, tokens_k=16), L.ERR_UNSUPPORTED),              # 2^31 heads
    (dict(tokens_k=(1 << 31) - 1), L.ERR_UNSUPPORTED)])
def test_decode_counts_heads_not_places(kw, status):
    """A missing workspace is what ends the calls that are accepted; those that need none are given one that lies on q."""
    d = decode_desc(lse=None, lengths=None, workspace=None, workspace_bytes=0, **kw)
    hd, h, hkv, places = d.head_dim, d.heads, d.kv_heads, d.tokens_k
    at = 1 << 44
    for name, n, strides in (("q", h, (h * hd, 0, hd)), ("out", h, (h * hd, 0, hd)), ("k", hkv, (places * hkv * hd, hkv * hd, hd)),
                             ("v", hkv, (places * hkv * hd, hkv * hd, hd))):
        setattr(d, name, view(at, *strides))
        at += 1 << 42
    need = L.lib().llmt_b200_attention_window_decode_workspace_bytes(ctypes.byref(d))
    if status == L.ERR_WORKSPACE and need == 0:
        d.lse, status = d.q.data, L.ERR_INVALID
    assert L.lib().llmt_b200_attention_window_decode(ctypes.byref(d), None) == status, L.last_error()


class _Tensor:
    """What the native functions look at of a tensor."""
    def __init__(self, at, dtype, *shape, stride=None):
        t = torch.empty(shape, dtype=dtype, device="meta")
        self.at, self.dtype, self.shape, self.nbytes, self.strides = at, dtype, t.shape, t.numel() * t.element_size(), stride or t.stride()

    def data_ptr(self):
        return self.at

    def stride(self):
        return self.strides

    def get_device(self):
        return 0


@pytest.mark.parametrize("name", ["norm_residual_bwd", "attention_window_fwd", "attention_window_bwd", "attention_window_decode"])
def test_a_workspace_of_bytes_stays_on_the_native_path(name):
    """The native function with what torch would tell it of a GPU, and addresses that the library refuses: its own message comes
    back, and the Python function is not asked."""
    code = ("import sys, ctypes, pytest, torch, llmt_b200 as L\n"
            "from llmt_b200 import _native\n"
            "from tests.test_block_ops_edges_cpu import MB, _Tensor as T\n"
            "name = sys.argv[1]\n"
            "asked = []\n"
            "exec(f'def {name}(*a, **k): asked.append(1)')\n"
            "bind = lambda: _native.bind(tuple(ctypes.cast(getattr(L.lib(), 'llmt_b200_' + n), ctypes.c_void_p).value for n in _native.NAMES),\n"
            "                            lambda d: 0, lambda: 0, torch.float32, torch.bfloat16, torch.int32, torch.float64, L.GemmDesc)\n"
            "_native.setup(bind, L._check, L._scratch)\n"
            "native = _native.fast(locals()[name])\n"
            "bf, f32 = torch.bfloat16, torch.float32\n"
            "q, k = (lambda i: T(i * MB, bf, 1, 64, 2, 64)), (lambda i: T(i * MB, bf, 1, 8192, 1, 64))\n"
            "token, lse = (lambda i: T(i * MB, bf, 2, 64, 64)), T(20 * MB, f32, 1, 2, 64)\n"
            "cache = lambda i: T(i * MB, bf, 2, 65536, 1, 64)\n"
            "row, w = (lambda i: T(i * MB, f32, 64, 64)), (lambda i: T(i * MB, f32, 64))\n"
            "calls = dict(norm_residual_bwd=lambda **ws: native(row(1), None, None, row(2), row(3), w_pre=w(4), rstd_pre=w(5), dw_pre=w(6), **ws),\n"
            "             attention_window_fwd=lambda **ws: native(q(1), lse, q(2), k(3), k(6), **ws),\n"
            "             attention_window_bwd=lambda **ws: native(q(1), k(3), k(6), q(2), q(9), k(10), k(13), q(16), lse, **ws),\n"
            "             attention_window_decode=lambda **ws: native(token(1), token(2), cache(100), cache(200), **ws))\n"
            "with pytest.raises(L.LlmtB200Error, match='16-byte aligned'):\n"
            "    calls[name](workspace=T(300 * MB + 8, torch.uint8, 64 * MB))\n"
            "assert not asked\n"
            "calls[name](workspace=T(300 * MB, torch.uint8, 64 * MB, stride=(0,)))\n"
            "assert asked, 'one that is not contiguous is'\n")
    subprocess.check_call([sys.executable, "-c", code, name], cwd=ROOT)


def test_python_refuses_rows_without_columns():
    x, w = torch.zeros(4, 0), torch.zeros(0)
    for call in (lambda: L.norm_residual_fwd(x, x, x, x, gate=torch.zeros(1, 0), w_pre=w),
                 lambda: L.norm_residual_bwd(x, x, x, x, x, x, gate=torch.zeros(1, 0), dgate=torch.zeros(1, 0), w_pre=w)):
        with pytest.raises(L.LlmtB200Error):
            call()


@pytest.mark.parametrize("name", ["norm_residual_bwd", "attention_window_fwd", "attention_window_bwd", "attention_window_decode"])
def test_a_call_reads_the_budget_of_sms_once(name):
    """The workspace that is asked for and the plan that is run are of one reading: the budget is the process's, and calls for
    another device may be under way while it is set."""
    source = open(os.path.join(ROOT, "llmt_b200", "csrc", "capi.cu")).read()
    body = source[source.index(f"int llmt_b200_{name}(const"):]
    body = re.sub(r"//[^\n]*", "", body[:body.index("\n}\n")])
    assert len(re.findall(r"\bsm_count\(\)|\bnorm_residual_plan_of\(|_workspace_bytes\(d\)", body)) == 1
