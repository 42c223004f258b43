"""What the block operators of llmt's C++ interface answer without a GPU."""
import ctypes
import os
import signal
import subprocess

import pytest

import llmt_b200 as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "_build", "test_block_ops_host")


def run(*args):
    assert os.path.exists(BIN), "run `python -m llmt_b200.build` (or __graft_entry__.build()) first"
    return subprocess.run([BIN, *map(str, args)], capture_output=True, text=True, timeout=60)


@pytest.mark.parametrize("b,t,h,hkv,hd,window,sinks", [(1, 8192, 2, 2, 64, 2048, 4), (1, 8192, 1, 1, 128, 0, 0), (8, 1024, 12, 12, 64, 256, 4),
                                                       (1, 300, 4, 2, 64, 0, 0), (2, 4096, 1, 1, 64, 0, 0)])
def test_attention_workspace_is_enough_for_either_direction(b, t, h, hkv, hd, window, sinks):
    d = L.AttentionDesc()
    d.batch, d.heads, d.kv_heads, d.tokens_q, d.tokens_k, d.head_dim, d.window, d.sinks, d.scale, d.dtype = b, h, hkv, t, t, hd, window, sinks, 1.0, L.BF16
    fwd, bwd = (int(getattr(L.lib(), f"llmt_b200_attention_window_{n}workspace_bytes")(ctypes.byref(d))) for n in ("fwd_", ""))
    r = run("workspace", b, t, h, hkv, hd, window, sinks)
    assert r.returncode == 0 and [int(x) for x in r.stdout.split()] == [max(fwd, bwd), fwd]


def test_rows_without_columns_are_refused_with_a_message():
    r = run("norm", 4, 0)
    assert r.returncode == -signal.SIGABRT and "[llmt] norm_residual_fwd" in r.stderr and "bad shape" in r.stderr
