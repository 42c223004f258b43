"""Attention with a sliding window and sinks, against the formulas in 64 bits and against differences."""
import math

import pytest

torch = pytest.importorskip("torch")

import llmt_b200 as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
# A probability (or dS) that is an operand is rounded to bf16: half a step, 2^-8.  Before that it carries the score's fp32
# error: 128 products of sums |q| |k| scale of up to 100 give 128 * 100 * 2^-24 < 2^-10, the exponential less.
P = 2.0 ** -8 + 2.0 ** -10


def _visible(tq, tk, window, sinks):
    p = torch.arange(tq, device=DEV)[:, None] + tk - tq
    j = torch.arange(tk, device=DEV)[None]
    seen = j <= p
    if window > 0:
        seen &= (j > p - window) | (j < sinks)
    return seen


def _heads(x, h):
    """[B, T, Hkv, hd] as fp64 [B, H, T, hd]."""
    return x.double().repeat_interleave(h // x.shape[2], 2).transpose(1, 2)


def _forward(q, k, v, window, sinks, scale=None):
    h = q.shape[2]
    q, k, v = (_heads(x, h) for x in (q, k, v))
    seen = _visible(q.shape[2], k.shape[2], window, sinks)
    s = (q @ k.transpose(-1, -2)) * (scale or q.shape[-1] ** -0.5)
    s = torch.where(seen, s, -math.inf)
    m = s.amax(-1, keepdim=True) if s.shape[-1] else torch.full((*s.shape[:-1], 1), -math.inf, device=DEV, dtype=torch.float64)
    e = torch.where(seen, (s - torch.where(m.isinf(), 0, m)).exp(), 0)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1, total)
    lse = torch.where(total == 0, -math.inf, m + total.log())[..., 0]
    return p, lse, p @ v, p @ v.abs()


def _check_forward(out, lse, q, k, v, window, sinks, scale=None):
    _, want_lse, want, size = _forward(q, k, v, window, sinks, scale)
    got = out.double().transpose(1, 2)
    # the result's rounding, and the probabilities' as operands
    bound = want.abs() * 2.0 ** -8 + size * P
    assert bool(((got - want).abs() <= bound + 1e-30).all()), float(((got - want).abs() / (bound + 1e-30)).max())
    empty = want_lse == -math.inf
    assert bool((lse[empty] == -math.inf).all()) and bool((got[empty] == 0).all())
    # scores' errors as in P, the logarithm's and the sum's roundings relative to values of up to 16
    assert bool(((lse.double() - want_lse).abs()[~empty] <= 2.0 ** -10 + 16 * 2.0 ** -22).all())


def _check_backward(dq, dk, dv, dout, q, k, v, out, lse, window, sinks, scale=None):
    """Against the formulas on what the call read: lse as stored, and out for queries that may see more than 128 keys."""
    b, tq, h, hd = q.shape
    hkv, tk = k.shape[2], k.shape[1]
    c = scale or hd ** -0.5
    seen = _visible(tq, tk, window, sinks)
    qd, kd, vd, od, dod = (_heads(x, h) for x in (q, k, v, out, dout))
    p = torch.where(seen, (qd @ kd.transpose(-1, -2) * c - lse.double()[..., None]).exp(), 0)
    dp, d = dod @ vd.transpose(-1, -2), (dod * od).sum(-1, keepdim=True)
    if min(window + sinks if window > 0 else tk, tk) <= 128:
        d = (p * dp).sum(-1, keepdim=True)
    ds = torch.where(seen, p * (dp - d), 0)
    # dK is formed with the row sums of P dP, which are D but for the rounding of out
    ds_k = torch.where(seen, p * (dp - (p * dp).sum(-1, keepdim=True)), 0)
    # dS: its rounding as an operand and P's relative error, fp32 products of hd terms in dP and D
    off = P * torch.maximum(ds.abs(), ds_k.abs()) + p * hd * 2.0 ** -23 * (dod.abs() @ vd.abs().transpose(-1, -2) + (dod * od).abs().sum(-1, keepdim=True))

    def group(x):
        return x.reshape(b, hkv, h // hkv, x.shape[-2], hd).sum(2).transpose(1, 2)
    for name, got, want, bound in (("dq", dq, (c * ds @ kd).transpose(1, 2), (c * off @ kd.abs()).transpose(1, 2)),
                                   ("dk", dk, group(c * ds_k.transpose(-1, -2) @ qd), group(c * off.transpose(-1, -2) @ qd.abs())),
                                   ("dv", dv, group(p.transpose(-1, -2) @ dod), group(P * p.transpose(-1, -2) @ dod.abs()))):
        # accumulation in fp32, truncated by the tensor cores, of at most 4096 terms: 2^-11 of the terms' sizes
        bound = want.abs() * 2.0 ** -8 + bound * (1 + 2.0 ** -3) + 1e-30
        assert bool(((got.double() - want).abs() <= bound).all()), f"{name}: {float(((got.double() - want).abs() / bound).max()):.2f} of the bound"


def _make(b, h, hkv, tq, tk, hd, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + tq * 31 + tk)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g).to(BF)
    return n(b, tq, h, hd), n(b, tk, hkv, hd), n(b, tk, hkv, hd), n(b, tq, h, hd)


CASES = [  # b, h, hkv, tq, tk, hd, window, sinks
    (1, 1, 1, 1, 1, 8, 0, 0), (2, 2, 1, 3, 3, 32, 2, 0), (1, 3, 3, 64, 64, 64, 0, 0), (1, 2, 2, 127, 127, 64, 17, 3), (1, 2, 1, 128, 128, 128, 64, 1),
    (2, 4, 2, 129, 129, 64, 128, 4), (1, 1, 1, 300, 300, 72, 1, 0), (1, 2, 1, 333, 333, 128, 100, 130), (1, 6, 2, 257, 257, 96, 0, 0),
    (1, 2, 2, 700, 700, 64, 129, 5), (1, 1, 1, 700, 700, 128, 64, 64), (2, 2, 1, 1, 500, 64, 0, 0), (1, 2, 1, 70, 500, 128, 90, 4), (1, 2, 1, 200, 1031, 64, 600, 260),
    (1, 1, 1, 40, 20, 64, 0, 0), (1, 2, 2, 300, 150, 128, 40, 2), (1, 1, 1, 260, 5, 64, 3, 1), (3, 3, 1, 65, 65, 40, 1000, 9), (1, 4, 1, 1025, 1025, 64, 256, 4),
    (1, 1, 1, 512, 512, 16, 512, 512), (1, 1, 1, 1500, 1500, 128, 0, 0),
]


@pytest.mark.parametrize("b,h,hkv,tq,tk,hd,window,sinks", CASES)
def test_forward_and_backward(b, h, hkv, tq, tk, hd, window, sinks):
    q, k, v, dout = _make(b, h, hkv, tq, tk, hd)
    out, lse = torch.full_like(q, 7.0), torch.full((b, h, tq), 7.0, device=DEV)
    L.attention_window_fwd(out, lse, q, k, v, window, sinks)
    assert L.device_status() == (0, 0)
    _check_forward(out, lse, q, k, v, window, sinks)
    dq, dk, dv = torch.full_like(q, 7.0), torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    L.attention_window_bwd(dq, dk, dv, dout, q, k, v, out, lse, window, sinks)
    assert L.device_status() == (0, 0)
    _check_backward(dq, dk, dv, dout, q, k, v, out, lse, window, sinks)
    again = [torch.empty_like(x) for x in (out, dq, dk, dv)]
    L.attention_window_fwd(again[0], lse, q, k, v, window, sinks)
    L.attention_window_bwd(*again[1:], dout, q, k, v, out, lse, window, sinks)
    assert all(torch.equal(x, y) for x, y in zip(again, (out, dq, dk, dv))), "the same bits on every run"


@pytest.mark.parametrize("hd", [64, 128])
def test_packed_projection_and_head_major_layouts(hd):
    b, h, hkv, t = 2, 4, 2, 200
    q, k, v, dout = _make(b, h, hkv, t, t, hd)
    want = [torch.empty_like(q), torch.empty(b, h, t, device=DEV), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]
    L.attention_window_fwd(*want[:2], q, k, v, 70, 4, scale=0.2)
    L.attention_window_bwd(*want[2:], dout, q, k, v, *want[:2], 70, 4, scale=0.2)
    packed = torch.cat((q, k, v, torch.full_like(k, 9.0)), 2)
    cut = lambda x: (x[:, :, :h], x[:, :, h:h + hkv], x[:, :, h + hkv:h + 2 * hkv])
    grads = torch.full_like(packed, 5.0)
    out, lse = torch.empty(b, h, t, hd, device=DEV, dtype=BF).transpose(1, 2), torch.empty(b, h, t, device=DEV)
    L.attention_window_fwd(out, lse, *cut(packed), 70, 4, scale=0.2)
    L.attention_window_bwd(*cut(grads), dout, *cut(packed), out, lse, 70, 4, scale=0.2)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert all(torch.equal(x, y) for x, y in zip(cut(grads), want[2:]))
    assert bool((grads[:, :, h + 2 * hkv:] == 5.0).all()), "what lies beside the gradients stays"


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), torch.finfo(BF).min])
def test_hidden_places_reach_nothing(hd, bad):
    """Right padding of a batch: the rows in front of it are those of the same call with zeros behind."""
    b, h, hkv, t, real, window, sinks = 1, 2, 1, 300, 150, 40, 3
    q, k, v, dout = _make(b, h, hkv, t, t, hd)
    dout[:, real:] = 0
    got = []
    for fill in (0.0, bad):
        for x in (q, k, v):
            x[:, real:] = fill
        out, lse = torch.empty_like(q), torch.empty(b, h, t, device=DEV)
        L.attention_window_fwd(out, lse, q, k, v, window, sinks)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        o2, l2 = out.clone(), lse.clone()
        o2[:, real:], l2[:, :, real:] = 0, 0   # what a user masks of the padding
        seen = dict(window=window, sinks=sinks)
        L.attention_window_bwd(dq, dk, dv, dout, q, k, v, o2, l2, **seen)
        got.append((out[:, :real].double(), lse[:, :, :real].double(), dq[:, :real].double()))
    assert L.device_status() == (0, 0)
    for x, y in zip(*got):
        assert bool(torch.isfinite(y).all())
        # one side may take another order of additions: the bounds of either
        assert float((x - y).norm()) <= 2 * P * float(x.norm())


@pytest.mark.parametrize("where", ["v", "k", "q", "dout"])
def test_a_value_that_is_not_finite_reaches_those_that_see_it(where):
    b, h, hkv, t, hd, window, sinks, at = 1, 1, 1, 200, 64, 30, 2, 100
    q, k, v, dout = _make(b, h, hkv, t, t, hd)
    dict(q=q, k=k, v=v, dout=dout)[where][0, at, 0, 5] = float("nan")
    out, lse = torch.empty_like(q), torch.empty(b, h, t, device=DEV)
    L.attention_window_fwd(out, lse, q, k, v, window, sinks)
    sees = torch.zeros(t, dtype=torch.bool, device=DEV)
    if where in "vk":
        sees[at:at + window] = True
    elif where == "q":
        sees[at] = True
    assert bool((torch.isnan(out[0, :, 0]).any(-1) == sees).all())
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    L.attention_window_bwd(dq, dk, dv, dout, q, k, v, out, lse, window, sinks)
    queries = sees.clone()
    if where == "dout":
        queries[at] = True
    assert bool((torch.isnan(dq[0, :, 0]).any(-1) == queries).all())
    keys = (_visible(t, t, window, sinks) & queries[:, None]).any(0)
    assert bool((torch.isnan(dk[0, :, 0]).any(-1) == keys).all())


def test_gradients_match_differences():
    b, h, hkv, t, hd, window, sinks = 1, 2, 1, 90, 32, 20, 3
    q, k, v, dout = _make(b, h, hkv, t, t, hd)
    out, lse = torch.empty_like(q), torch.empty(b, h, t, device=DEV)
    L.attention_window_fwd(out, lse, q, k, v, window, sinks)
    g = dict(q=torch.empty_like(q), k=torch.empty_like(k), v=torch.empty_like(v))
    L.attention_window_bwd(g["q"], g["k"], g["v"], dout, q, k, v, out, lse, window, sinks)
    x = dict(q=q, k=k, v=v)
    for name, grad in g.items():
        way = torch.randn(x[name].shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
        e = 2.0 ** -4
        ends, moved = [], []
        for sign in (1, -1):
            y = {**x, name: (x[name].float() + sign * e * way).to(BF)}
            o = torch.empty_like(q)
            L.attention_window_fwd(o, None, y["q"], y["k"], y["v"], window, sinks)
            ends.append((o.double() * dout.double()).sum())
            moved.append(y[name].double())
        slope = (grad.double() * (moved[0] - moved[1])).sum()
        # out is rounded (2^-8 relative, at random over thousands of terms: 6 deviations of 2^-9) at both ends, the third-order
        # term is e^2 / 6 of the slope's terms, grad is rounded too
        noise = 6 * 2.0 ** -9 * 2 ** 0.5 * float((out.double() * dout.double()).norm())
        slack = (e * e + 4 * 2.0 ** -9) * float((grad.double() * (moved[0] - moved[1])).norm()) * 6
        assert abs(float(ends[0] - ends[1] - slope)) <= noise + slack, name


@pytest.mark.parametrize("b,h,hkv,cap,hd,window,sinks", [(1, 1, 1, 1, 8, 0, 0), (3, 4, 2, 77, 64, 0, 0), (4, 12, 12, 400, 64, 64, 4), (5, 8, 1, 1000, 128, 300, 130),
                                                         (2, 32, 8, 5000, 128, 0, 0), (7, 6, 3, 259, 72, 1, 0), (1, 40, 2, 130, 96, 50, 60), (2, 3, 1, 2050, 40, 2000, 7)])
def test_decode(b, h, hkv, cap, hd, window, sinks):
    g = torch.Generator(device=DEV).manual_seed(cap)
    q = torch.randn(b, h, hd, device=DEV, generator=g).to(BF)
    k, v = (torch.randn(b, cap, hkv, hd, device=DEV, generator=g).to(BF) for _ in "kv")
    lengths = torch.randint(1, cap + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
    lengths[0] = cap
    if b > 2:
        lengths[1], lengths[2] = 0, 1
    for i, n in enumerate(lengths.tolist()):   # places behind a sequence hold anything
        k[i, n:], v[i, n:] = float("nan"), float("inf")
    out, lse = torch.full_like(q, 7.0), torch.full((b, h), 7.0, device=DEV)
    L.attention_window_decode(out, q, k, v, lengths, window, sinks, lse=lse)
    for i, n in enumerate(lengths.tolist()):
        if n == 0:
            assert bool((out[i] == 0).all()) and bool((lse[i] == -math.inf).all())
            continue
        _check_forward(out[i][None, None], lse[i][None, :, None], q[i][None, None], k[i:i + 1, :n], v[i:i + 1, :n], window, sinks)
    if b == 1 or not bool(torch.isnan(k).any()):
        o2 = torch.empty_like(out)
        L.attention_window_decode(o2, q, k, v, None, window, sinks)
        assert torch.equal(o2, out)
    past = torch.full_like(lengths, cap + 100)
    full_k, full_v = torch.nan_to_num(k, nan=0.5, posinf=0.5), torch.nan_to_num(v, nan=0.5, posinf=0.5)
    o3, o4 = torch.empty_like(out), torch.empty_like(out)
    L.attention_window_decode(o3, q, full_k, full_v, past, window, sinks)
    L.attention_window_decode(o4, q, full_k, full_v, None, window, sinks)
    assert torch.equal(o3, o4), "a length past the cache counts as the cache"


def test_another_stream_and_a_captured_step():
    b, h, hkv, t, hd = 1, 4, 2, 300, 64
    q, k, v, dout = _make(b, h, hkv, t, t, hd)
    out, lse, dq, dk, dv = torch.empty_like(q), torch.empty(b, h, t, device=DEV), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws = torch.empty(L.attention_window_workspace_bytes(q, k, 64, 4), dtype=torch.uint8, device=DEV)

    def step(stream=None):
        L.attention_window_fwd(out, lse, q, k, v, 64, 4, stream=stream)
        L.attention_window_bwd(dq, dk, dv, dout, q, k, v, out, lse, 64, 4, workspace=ws, stream=stream)
    step()
    want = [x.clone() for x in (out, dq, dk, dv)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for x in (out, dq, dk, dv):
        x.zero_()
    side.wait_stream(torch.cuda.current_stream())
    step(side)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip((out, dq, dk, dv), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for x in (out, dq, dk, dv):
        x.zero_()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip((out, dq, dk, dv), want))
    del graph


def test_nothing_to_do():
    e = torch.empty(0, 5, 2, 64, device=DEV, dtype=BF)
    L.attention_window_fwd(e, None, e, e, e)
    q, k = torch.ones(1, 5, 2, 64, device=DEV, dtype=BF), torch.empty(1, 0, 2, 64, device=DEV, dtype=BF)
    out, lse = torch.full_like(q, 3.0), torch.zeros(1, 2, 5, device=DEV)
    L.attention_window_fwd(out, lse, q, k, k)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq = torch.full_like(q, 3.0)
    L.attention_window_bwd(dq, k.clone(), k.clone(), q, q, k, k, out, lse)
    assert bool((dq == 0).all())
    none = torch.empty(1, 0, 2, 64, device=DEV, dtype=BF)
    dk, dv = torch.full_like(q, 3.0), torch.full_like(q, 3.0)
    L.attention_window_bwd(none, dk, dv, none.clone(), none.clone(), q, q.clone(), none.clone(), torch.empty(1, 2, 0, device=DEV))
    assert bool((dk == 0).all()) and bool((dv == 0).all())
