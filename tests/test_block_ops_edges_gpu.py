"""Rotary positions, norms around a block and windowed attention at the edge of what their header allows."""
import pytest

torch = pytest.importorskip("torch")

import llmt_b200 as L
from tests.test_attention_window_gpu import _make
from tests.test_norm_residual_gpu import _close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def test_attention_without_query_heads_zeroes_the_key_gradients():
    q = torch.empty(2, 5, 0, 64, device=DEV, dtype=BF)
    k, v = torch.ones(2, 7, 3, 64, device=DEV, dtype=BF), torch.ones(2, 7, 3, 64, device=DEV, dtype=BF)
    dk, dv, lse = torch.full_like(k, 3.0), torch.full_like(v, 3.0), torch.empty(2, 0, 5, device=DEV)
    L.attention_window_fwd(q.clone(), lse, q, k, v)
    L.attention_window_bwd(q.clone(), dk, dv, q.clone(), q, k, v, q.clone(), lse)
    assert bool((dk == 0).all()) and bool((dv == 0).all())


@pytest.mark.parametrize("cols", [64, 61])
def test_norm_gradients_of_rows_of_any_size(cols):
    """Rows so small or large that a power of their rstd leaves fp32's range, while every result is inside it."""
    g = torch.Generator(device=DEV).manual_seed(cols)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g)
    out_size = torch.tensor([0, 0, 0, -62, 58, -30, 0, 20], device=DEV)[:, None]
    y_size = torch.tensor([0, -46, 52, 0, 0, 30, -60, -20], device=DEV)[:, None]
    rows = out_size.shape[0]
    out, y = n(rows, cols) * 2.0 ** out_size, n(rows, cols) * 2.0 ** y_size
    dout, dh, w_post, w_pre = n(rows, cols), 16 * n(rows, cols), 1 + 0.1 * n(cols), 1 + 0.1 * n(cols)
    rs, rp = (z.double().square().mean(-1).rsqrt().float() for z in (out, y))
    dx, dy, dw_post, dw_pre = torch.empty_like(out), torch.empty_like(y), torch.empty(cols, device=DEV), torch.empty(cols, device=DEV)
    L.norm_residual_bwd(dx, dy, dout, dh, out, y, w_post=w_post, w_pre=w_pre, rstd_post=rp, rstd_pre=rs, dw_post=dw_post, dw_pre=dw_pre)
    r, a, k, c = rs.double()[:, None], dh.double() * w_pre.double(), w_post.double(), y.double() * rp.double()[:, None]
    b, mean = out.double() * r, lambda t: t.mean(-1, keepdim=True)
    gx, size = dout.double() + r * (a - b * mean(a * b)), dout.double().abs() + r * (a.abs() + b.abs() * mean((a * b).abs()))
    # the roundings are counted as in tests/test_norm_residual_gpu.py: products and the sums of a row's terms
    _close(dx, gx, 64, size, "dx")
    q = rp.double()[:, None]
    _close(dy, q * (k * gx - c * mean(k * gx * c)), 160, q * (k.abs() * size + c.abs() * mean(k.abs() * size * c.abs())), "dy")
    _close(dw_pre, (dh.double() * b).sum(0), 100, (dh.double() * b).abs().sum(0), "dw_pre")
    _close(dw_post, (gx * c).sum(0), 200, (size * c.abs()).sum(0), "dw_post")


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_norm_gradient_of_a_block_without_a_norm_does_not_depend_on_it(bad):
    rows, cols = 5, 40
    g = torch.Generator(device=DEV).manual_seed(1)
    dout, y, gate = (torch.randn(rows, cols, device=DEV, generator=g) for _ in range(3))
    dx, dy, dgate, want = (torch.empty_like(y) for _ in range(4))
    L.norm_residual_bwd(dx, want, dout, None, None, y, gate=gate, dgate=dgate, scale=0.5)
    y[2, 7] = bad
    L.norm_residual_bwd(dx, dy, dout, None, None, y, gate=gate, dgate=dgate, scale=0.5)
    assert torch.equal(dx, dout) and torch.equal(dy, want)
    there = torch.isfinite(dgate)   # the gate's gradient is g y
    assert not bool(there[2, 7]) and int(there.sum()) == rows * cols - 1


@pytest.mark.parametrize("order", ["bhtd", "bthd", "thbd"])
def test_gradients_packed_in_any_order(order):
    """dq, dk and dv as views of one buffer, whatever the order of its dimensions."""
    b, h, hkv, t, hd, window, sinks = 2, 4, 2, 130, 64, 50, 3
    q, k, v, dout = _make(b, h, hkv, t, t, hd)
    out, lse = torch.empty_like(q), torch.empty(b, h, t, device=DEV)
    L.attention_window_fwd(out, lse, q, k, v, window, sinks)
    want = [torch.empty_like(x) for x in (q, k, v)]
    L.attention_window_bwd(*want, dout, q, k, v, out, lse, window, sinks)
    n = dict(b=b, t=t, h=h + 2 * hkv + 1, d=hd)
    buffer = torch.full([n[x] for x in order], 5.0, device=DEV, dtype=BF)
    grads = buffer.permute(*(order.index(x) for x in "bthd"))
    parts = grads[:, :, :h], grads[:, :, h:h + hkv], grads[:, :, h + hkv:h + 2 * hkv]
    L.attention_window_bwd(*parts, dout, q, k, v, out, lse, window, sinks)
    assert all(torch.equal(x, y) for x, y in zip(parts, want))
    assert bool((grads[:, :, h + 2 * hkv:] == 5.0).all()), "what lies beside the gradients stays"


def test_rope_between_the_rows_that_it_reads():
    """The turned heads beside the plain ones in one token row."""
    g = torch.Generator(device=DEV).manual_seed(4)
    rows = torch.randn(2, 9, 6, 32, device=DEV, generator=g).to(BF)
    freqs = L.rope_frequencies(32, device=DEV)
    want, before = torch.empty(2, 9, 3, 32, device=DEV, dtype=BF), rows.clone()
    L.rope(want, rows[:, :, :3], freqs, offset=5)
    L.rope(rows[:, :, 3:], rows[:, :, :3], freqs, offset=5)
    assert torch.equal(rows[:, :, 3:], want) and torch.equal(rows[:, :, :3], before[:, :, :3])


def test_norm_rows_beside_one_another():
    """The residual stream, its sum with the block and the normed rows as columns of one buffer."""
    rows, c = 13, 24
    g = torch.Generator(device=DEV).manual_seed(5)
    buffer = torch.randn(rows, 4 * c, device=DEV, generator=g)
    x, y, out, h = (buffer[:, i * c:(i + 1) * c] for i in range(4))
    w = torch.ones(c, device=DEV)
    want, before = (torch.empty(rows, c, device=DEV), torch.empty(rows, c, device=DEV)), buffer.clone()
    L.norm_residual_fwd(*want, x.contiguous(), y.contiguous(), w_pre=w)
    L.norm_residual_fwd(out, h, x, y, w_pre=w)
    assert torch.equal(out, want[0]) and torch.equal(h, want[1]) and torch.equal(buffer[:, :2 * c], before[:, :2 * c])
