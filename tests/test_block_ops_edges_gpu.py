"""Rotary positions, norms around a block and windowed attention at the edge of what their header allows."""
import math

import pytest

torch = pytest.importorskip("torch")

import llmt_b200 as L
from tests.test_attention_window_gpu import P, _check_forward, _heads, _make, _visible
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


def _summed(seen, f, x):
    """Sum over the second-last dimension of x of f[..., i, j] x[..., j, :], visible pairs only (0 * inf of the others apart)."""
    return torch.where(seen[..., None], f[..., None] * x[..., None, :, :], 0).sum(-2)


def _same_kind(got, want, bound, what):
    """NaN and infinity where the definition has them, the others within the bound (nothing is asked where that has no size)."""
    assert bool((torch.isnan(got) == torch.isnan(want)).all()), f"{what}: NaN at {int((torch.isnan(got) != torch.isnan(want)).sum())} other places"
    inf = torch.isinf(want)
    assert bool((torch.isinf(got) == inf).all()) and bool((got[inf] == want[inf]).all()), f"{what}: infinities"
    off, finite = (got - want).abs(), torch.isfinite(want) & torch.isfinite(bound)
    assert bool((off[finite] <= bound[finite]).all()), f"{what}: {float((off[finite] / bound[finite]).max()):.2f} of the bound"


SPOILT = [(n, how, bad) for n in ("q", "k", "v", "dout") for how in ("column", "one", "some") for bad in (math.nan, math.inf, -math.inf)]


@pytest.mark.parametrize("b,h,hkv,tq,tk,hd,window,sinks", [
    (1, 2, 1, 200, 200, 64, 30, 2),       # a short window: D summed exactly
    (1, 2, 2, 260, 260, 128, 0, 0),
    (1, 2, 1, 40, 1300, 64, 700, 3),      # in parts
    (1, 4, 2, 150, 100, 72, 0, 0),        # queries that see nothing
    (1, 4, 1, 700, 700, 64, 0, 0),        # dK and dV in parts
    (1, 2, 1, 600, 600, 128, 100, 130)])  # sinks of two tiles
def test_values_that_are_not_finite_reach_what_the_definition_says(b, h, hkv, tq, tk, hd, window, sinks):
    """A weight, a token or some values that are NaN or infinite, and hidden places that hold infinities beside them."""
    g = torch.Generator(device=DEV).manual_seed(9)
    seen, c = _visible(tq, tk, window, sinks), hd ** -0.5
    for name, how, bad in SPOILT:
        q, k, v, dout = _make(b, h, hkv, tq, tk, hd)
        x = dict(q=q, k=k, v=v, dout=dout)[name]
        if how == "column":
            x[..., 5] = bad
        elif how == "one":
            x[0, x.shape[1] * 2 // 3, 0, 3] = bad
        else:
            at = torch.randint(0, x.numel(), (3,), device=DEV, generator=g)
            x.view(-1)[at] = torch.tensor([bad, -bad, bad], device=DEV, dtype=BF)
        hidden = ~seen.any(0)
        k[:, hidden], v[:, hidden] = math.inf, -math.inf
        out, lse = torch.empty_like(q), torch.empty(b, h, tq, device=DEV)
        L.attention_window_fwd(out, lse, q, k, v, window, sinks)
        qd, kd, vd, dod = (_heads(y, h) for y in (q, k, v, dout))
        s = torch.where(seen, qd @ kd.transpose(-1, -2) * c, -math.inf)
        m = s.amax(-1, keepdim=True)
        e = (s - torch.where(m == -math.inf, 0, m)).exp()
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total == 0, 1, total)
        what = f"{name} {how} {bad}"
        want = _summed(seen, p, vd)
        _same_kind(out.double().transpose(1, 2), want, want.abs() * 2.0 ** -8 + _summed(seen, p, vd.abs()) * P + 1e-30, what + ": out")
        want_lse = torch.where(total == 0, -math.inf, m + total.log())[..., 0]
        _same_kind(lse.double(), want_lse, torch.full_like(want_lse, 2.0 ** -10 + 16 * 2.0 ** -22), what + ": lse")

        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        L.attention_window_bwd(dq, dk, dv, dout, q, k, v, out, lse, window, sinks)
        assert L.device_status() == (0, 0)
        ld, od = lse.double()[..., None], _heads(out, h)
        p = torch.where(seen, torch.where(ld == -math.inf, 0, (qd @ kd.transpose(-1, -2) * c - ld).exp()), 0)
        dp, by_rows = dod @ vd.transpose(-1, -2), torch.where(seen, p * (dod @ vd.transpose(-1, -2)), 0).sum(-1, keepdim=True)
        d = by_rows if min(window + sinks if window > 0 else tk, tk) <= 128 else (dod * od).sum(-1, keepdim=True)
        d_k = torch.where(torch.isfinite(by_rows), by_rows, d)
        ds, ds_k = (torch.where(seen, p * (dp - y), 0) for y in (d, d_k))
        off = P * torch.maximum(ds.abs(), ds_k.abs()) + p * hd * 2.0 ** -23 * (dod.abs() @ vd.abs().transpose(-1, -2) + (dod * od).abs().sum(-1, keepdim=True))

        def group(y):
            return y.reshape(b, hkv, h // hkv, tk, hd).sum(2).transpose(1, 2)
        t = seen.T
        for n, got, want, bound in (("dq", dq, _summed(seen, c * ds, kd).transpose(1, 2), _summed(seen, c * off, kd.abs()).transpose(1, 2)),
                                    ("dk", dk, group(_summed(t, c * ds_k.transpose(-1, -2), qd)), group(_summed(t, c * off.transpose(-1, -2), qd.abs()))),
                                    ("dv", dv, group(_summed(t, p.transpose(-1, -2), dod)), group(_summed(t, P * p.transpose(-1, -2), dod.abs())))):
            _same_kind(got.double(), want, want.abs() * 2.0 ** -8 + bound * (1 + 2.0 ** -3) + 1e-30, f"{what}: {n}")


def _time(call):
    """The least time of a few calls, in microseconds."""
    call()
    best = math.inf
    for _ in range(5):
        a, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        e.record()
        e.synchronize()
        best = min(best, 1e3 * a.elapsed_time(e))
    return best


@pytest.mark.parametrize("b,h,hkv,t,hd,window,sinks", [(1, 4, 2, 2048, 128, 0, 0), (2, 4, 4, 1024, 64, 256, 4)])
def test_a_step_whose_values_are_nan_takes_no_longer_than_a_few_others(b, h, hkv, t, hd, window, sinks):
    """Sixty times as long and more it took when every row that is NaN was summed again.  A token that is NaN still spoils the rows
    that share a tile with it and do not see it, 128 a head and pass at most: a warp has 32 of them in turn, and goes to memory
    for 32 places four times for their sums and for 16 places once to look at them, a microsecond each time at most."""
    def step(**spoil):
        x = dict(zip(("q", "k", "v", "dout"), _make(b, h, hkv, t, t, hd)))
        for name, where in spoil.items():
            x[name][where] = math.nan
        out, lse = torch.empty_like(x["q"]), torch.empty(b, h, t, device=DEV)
        dq, dk, dv = (torch.empty_like(x[n]) for n in "qkv")

        def call():
            L.attention_window_fwd(out, lse, x["q"], x["k"], x["v"], window, sinks)
            L.attention_window_bwd(dq, dk, dv, x["dout"], x["q"], x["k"], x["v"], out, lse, window, sinks)
        return _time(call)
    clean, column, token = step(), (Ellipsis, 5), (0, t // 2)
    for spoil in (dict(q=..., k=..., v=..., dout=...), dict(q=column), dict(k=column), dict(v=column), dict(dout=column), dict(q=token, k=token, v=token)):
        spoilt = step(**spoil)
        places = min(t, window + sinks) if window else t
        rows = 3 * 32 * (4 * places / 32 + places / 16) if token in spoil.values() else 0
        assert spoilt <= 10 * clean + rows, (spoil, clean, spoilt)


def test_decode_of_more_rows_than_an_index_counts():
    """256 sequences x 64 heads on 1 x 131072 places: 2^31 rows of all heads, 1 GB of keys and values; most places are empty."""
    b, h, places, hd = 256, 64, 131072, 8
    g = torch.Generator(device=DEV).manual_seed(8)
    q = torch.randn(b, h, hd, device=DEV, generator=g).to(BF)
    k, v = (torch.empty(b, places, 1, hd, device=DEV, dtype=BF) for _ in "kv")
    held = 70
    lengths = torch.randint(1, held + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
    lengths[-1] = places
    k[:, :held], v[:, :held] = (torch.randn(b, held, 1, hd, device=DEV, generator=g).to(BF) for _ in "kv")
    k[-1], v[-1] = (torch.randn(places, 1, hd, device=DEV, generator=g).to(BF) for _ in "kv")
    out = torch.full_like(q, 7.0)
    L.attention_window_decode(out, q, k, v, lengths)
    for i in (0, 1, 100, b - 2, b - 1):
        n = int(lengths[i])
        lse = torch.empty(1, h, 1, device=DEV)
        one = torch.empty(1, h, hd, device=DEV, dtype=BF)
        L.attention_window_decode(one, q[i:i + 1], k[i:i + 1], v[i:i + 1], lengths[i:i + 1], lse=lse.view(1, h))
        _check_forward(out[i][None, None], lse, q[i][None, None], k[i:i + 1, :n], v[i:i + 1, :n], 0, 0)
