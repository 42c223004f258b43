"""Attention of few queries over many keys, whose forward pass shares the keys of a query block out and joins the parts: against
the formulas in 64 bits, with hidden places that hold anything, with and without its workspace, and as the input of the
backward pass."""
import pytest

torch = pytest.importorskip("torch")

import llmt_b200 as L
from tests.test_attention_window_gpu import BF, DEV, _check_backward, _check_forward, _visible

pytestmark = pytest.mark.gpu

#        b  h hkv tq   tk    hd  window sinks
CASES = [(1, 2, 1, 64, 8192, 128, 0, 0),
         (1, 4, 2, 1, 4096, 64, 0, 0),
         (1, 1, 1, 300, 5000, 72, 0, 0),        # one head: two query blocks of it against the same keys
         (1, 4, 1, 200, 3001, 128, 2000, 130),  # sinks of two tiles, then a window that begins inside a tile
         (1, 3, 1, 257, 2999, 96, 700, 4),
         (2, 2, 1, 130, 2600, 64, 1500, 4),
         (1, 1, 1, 1500, 1400, 64, 0, 0),       # a hundred rows that see nothing
         (1, 2, 2, 1100, 1100, 128, 0, 0),      # parts of short rows are empty
         (1, 1, 1, 513, 4097, 8, 4000, 1)]


def _inputs(b, h, hkv, tq, tk, hd, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g).to(BF)
    return n(b, tq, h, hd), n(b, tk, hkv, hd), n(b, tk, hkv, hd), n(b, tq, h, hd)


def _results(q):
    return torch.full_like(q, float("nan")), torch.full((q.shape[0], q.shape[2], q.shape[1]), float("nan"), device=DEV)


@pytest.mark.parametrize("case", CASES, ids=str)
def test_parts_join_to_the_formula(case):
    b, h, hkv, tq, tk, hd, window, sinks = case
    q, k, v, dout = _inputs(b, h, hkv, tq, tk, hd)
    need = L.attention_window_fwd_workspace_bytes(q, k, window, sinks)
    assert need > 0, "the case is done in parts"
    out, lse = _results(q)
    L.attention_window_fwd(out, lse, q, k, v, window, sinks)
    _check_forward(out, lse, q, k, v, window, sinks)
    # with a workspace of the caller's: the same bits, and nothing behind it is touched
    ws = torch.full((need + 256,), 7, dtype=torch.uint8, device=DEV)
    again, lse2 = _results(q)
    L.attention_window_fwd(again, lse2, q, k, v, window, sinks, workspace=ws[:need])
    assert torch.equal(out, again) and torch.equal(lse, lse2) and bool((ws[need:] == 7).all())
    # with one that is too small: not in parts, right all the same
    whole, lse3 = _results(q)
    L.attention_window_fwd(whole, lse3, q, k, v, window, sinks, workspace=ws[:need - 16])
    _check_forward(whole, lse3, q, k, v, window, sinks)
    L.attention_window_fwd(again, None, q, k, v, window, sinks)
    assert torch.equal(out, again)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    L.attention_window_bwd(dq, dk, dv, dout, q, k, v, out, lse, window, sinks)
    _check_backward(dq, dk, dv, dout, q, k, v, out, lse, window, sinks)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), torch.finfo(BF).min])
@pytest.mark.parametrize("hd", [64, 128])
def test_hidden_places_reach_no_part(bad, hd):
    """Keys that a row does not see hold NaN, infinity or the lowest value: keys 4 .. 99 are hidden from every query, keys
    2000 .. 2049 from all but some."""
    b, h, hkv, tq, tk, window, sinks = 1, 2, 1, 90, 3000, 950, 4
    q, k, v, _ = _inputs(b, h, hkv, tq, tk, hd, seed=1)
    seen = _visible(tq, tk, window, sinks)[None, None]
    k[:, 4:100], v[:, 4:100] = bad, bad
    out, lse = _results(q)
    assert L.attention_window_fwd_workspace_bytes(q, k, window, sinks) > 0
    L.attention_window_fwd(out, lse, q, k, v, window, sinks)
    _check_forward(out, lse, q, k.masked_fill(k != k, 0).clamp(-8, 8), v.masked_fill(v != v, 0).clamp(-8, 8), window, sinks)
    v[:, 2000:2050] = bad
    L.attention_window_fwd(out, lse, q, k, v, window, sinks)
    clean = ~seen[0, 0, :, 2000:2050].any(-1)
    assert bool(clean.any()) and not bool(clean.all())
    part = out[:, clean].double()
    want, _ = _results(q)
    L.attention_window_fwd(want, None, q, k.masked_fill(k != k, 0).clamp(-8, 8), v.masked_fill(v != v, 0).clamp(-8, 8), window, sinks)
    # either side is off by the roundings of P and of the result
    assert bool(((part - want[:, clean].double()).abs() <= 2 * 2.0 ** -8 * (want[:, clean].double().abs() + 4)).all())
    if bad == bad and abs(bad) != float("inf"):
        return
    assert not bool(torch.isfinite(out[:, ~clean].float()).all(-1).any())


@pytest.mark.parametrize("bad", [float("nan"), float("-inf"), torch.finfo(BF).max])
@pytest.mark.parametrize("b,h,hkv,tq,tk,hd,window,sinks", [(1, 2, 1, 900, 4000, 128, 1500, 4), (1, 2, 2, 300, 2900, 64, 1200, 0), (1, 1, 1, 1300, 1200, 64, 0, 0)])
def test_gradients_of_parts(b, h, hkv, tq, tk, hd, window, sinks, bad):
    """dQ in parts (the workspace is larger than one whole pass wants), its share of D, and dK and dV after it, with keys that
    no query sees and queries that see nothing holding anything."""
    q, k, v, dout = _inputs(b, h, hkv, tq, tk, hd, seed=3)
    seen = _visible(tq, tk, window, sinks)
    hidden, idle = ~seen.any(0), ~seen.any(1)
    assert bool(hidden.any()) or bool(idle.any())
    ks, vs, qs, douts = k.clone(), v.clone(), q.clone(), dout.clone()
    for clean, spoilt, rows in ((k, ks, hidden), (v, vs, hidden), (q, qs, idle), (dout, douts, idle)):
        clean[:, rows], spoilt[:, rows] = 0, bad
    out, lse = _results(q)
    L.attention_window_fwd(out, lse, qs, ks, vs, window, sinks)
    _check_forward(out, lse, q, k, v, window, sinks)
    dq, dk, dv = (torch.full_like(x, float("nan")) for x in (q, k, v))
    L.attention_window_bwd(dq, dk, dv, douts, qs, ks, vs, out, lse, window, sinks)
    _check_backward(dq, dk, dv, dout, q, k, v, out, lse, window, sinks)
    assert bool((dk[:, hidden] == 0).all()) and bool((dv[:, hidden] == 0).all()) and bool((dq[:, idle] == 0).all())
    again = [torch.full_like(x, float("nan")) for x in (q, k, v)]
    L.attention_window_bwd(*again, douts, qs, ks, vs, out, lse, window, sinks)
    assert all(torch.equal(x, y) for x, y in zip(again, (dq, dk, dv)))


def test_parts_in_a_graph_and_on_another_stream():
    q, k, v, _ = _inputs(1, 2, 1, 64, 8192, 128, seed=2)
    out, lse = _results(q)
    L.attention_window_fwd(out, lse, q, k, v)
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.attention_window_fwd(out, lse, q, k, v)
    out.fill_(float("nan"))
    graph.replay()
    assert torch.equal(out, want)
    del graph
    side = torch.cuda.Stream()
    out.fill_(float("nan"))
    side.wait_stream(torch.cuda.current_stream())
    L.attention_window_fwd(out, lse, q, k, v, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)


def test_a_workspace_that_lies_on_a_tensor_is_refused():
    q, k, v, _ = _inputs(1, 2, 1, 64, 8192, 128)
    out, lse = _results(q)
    need = L.attention_window_fwd_workspace_bytes(q, k)
    ws = torch.empty(need + 16, dtype=torch.uint8, device=DEV)
    with pytest.raises(L.LlmtB200Error, match="16-byte aligned"):
        L.attention_window_fwd(out, lse, q, k, v, workspace=ws[8:8 + need])
    with pytest.raises(L.LlmtB200Error, match="overlaps lse"):
        L.attention_window_fwd(out, ws[256:256 + lse.numel() * 4].view(torch.float32).view(lse.shape), q, k, v, workspace=ws[:need])
