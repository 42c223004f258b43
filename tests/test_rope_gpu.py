"""Rotary positions against the formula in 64 bits."""
import math

import pytest

torch = pytest.importorskip("torch")

import llmt_b200 as L

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _reference(x, freqs, positions, interleaved, inverse, scale):
    x = x.double().clone()
    a = positions.double()[:, :, None, None] * freqs
    c, s = a.cos() * scale, a.sin() * (-scale if inverse else scale)
    r = 2 * freqs.numel()
    u, w = (x[..., 0:r:2].clone(), x[..., 1:r:2].clone()) if interleaved else (x[..., :r // 2].clone(), x[..., r // 2:r].clone())
    first, second = u * c - w * s, u * s + w * c
    if interleaved:
        x[..., 0:r:2], x[..., 1:r:2] = first, second
    else:
        x[..., :r // 2], x[..., r // 2:r] = first, second
    return x


def _close(y, ref, pair_norm):
    # Rounding of the result, and in fp32: cos and sin (2 ulp each), the frequency's product with scale, two products and a
    # sum, an angle resolved to 2^-32 turns: 8 roundings relative to the pair's length.
    half = torch.finfo(y.dtype).eps / 2
    bound = ref.abs() * half + pair_norm * 8 * 2.0 ** -24
    assert bool(((y.double() - ref).abs() <= bound).all()), float(((y.double() - ref).abs() - bound).max())


def _pair_norm(ref, r, interleaved):
    n = torch.zeros_like(ref)
    if interleaved:
        m = (ref[..., 0:r:2] ** 2 + ref[..., 1:r:2] ** 2).sqrt()
        n[..., 0:r:2] = n[..., 1:r:2] = m
    else:
        m = (ref[..., :r // 2] ** 2 + ref[..., r // 2:r] ** 2).sqrt()
        n[..., :r // 2] = n[..., r // 2:r] = m
    return n


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,t,heads,of,hd,rot", [(1, 1, 1, 1, 2, 2), (2, 5, 3, 3, 64, 64), (3, 17, 4, 6, 128, 64), (2, 9, 2, 3, 80, 20),
                                                 (1, 33, 5, 5, 7, 6), (2, 8, 3, 5, 256, 256), (1, 3, 2, 2, 16, 0)])
def test_rope(b, t, heads, of, hd, rot, dtype, interleaved):
    g = torch.Generator(device=DEV).manual_seed(b * 1000 + t)
    rows = torch.randn(b, t, of, hd, device=DEV, generator=g).to(dtype)
    x = rows[:, :, :heads]
    freqs = L.rope_frequencies(rot, factor=4.0, trained=1024.0, device=DEV)
    positions = torch.randint(-5, 2 ** 20, (b, t), device=DEV, generator=g, dtype=torch.int32)
    for inverse, scale in ((False, 1.0), (True, 1.3)):
        ref = _reference(x, freqs, positions, interleaved, inverse, scale)
        norm = _pair_norm(ref, rot, interleaved) if rot else torch.zeros_like(ref)
        y = torch.full_like(rows, 7.0)
        L.rope(y[:, :, :heads], x, freqs, positions, interleaved=interleaved, inverse=inverse, scale=scale)
        _close(y[:, :, :heads], ref, norm)
        assert bool((y[:, :, heads:] == 7.0).all()), "what is not rotated stays"
        here = rows.clone()
        L.rope(here[:, :, :heads], here[:, :, :heads], freqs, positions, interleaved=interleaved, inverse=inverse, scale=scale)
        assert torch.equal(here[:, :, :heads], y[:, :, :heads]) and torch.equal(here[:, :, heads:], rows[:, :, heads:])


def test_positions_by_offset_and_head_major_layout():
    b, t, h, hd = 2, 11, 3, 64
    x = torch.randn(b, h, t, hd, device=DEV).bfloat16().transpose(1, 2)
    freqs = L.rope_frequencies(hd, device=DEV)
    positions = (torch.arange(t, device=DEV, dtype=torch.int32) + 70000).expand(b, t).contiguous()
    y, z = torch.empty(b, t, h, hd, device=DEV, dtype=torch.bfloat16), torch.empty(b, t, h, hd, device=DEV, dtype=torch.bfloat16)
    L.rope(y, x, freqs, positions)
    L.rope(z, x, freqs, offset=70000)
    assert torch.equal(y, z)
    ref = _reference(x, freqs, positions, False, False, 1.0)
    _close(y, ref, _pair_norm(ref, hd, False))


def test_far_positions_keep_the_relative_angle():
    """The product of a rotated query and key depends on their distance alone, however far both are."""
    hd = 64
    freqs = L.rope_frequencies(hd, device=DEV)
    q, k = torch.randn(1, 1, 1, hd, device=DEV), torch.randn(1, 1, 1, hd, device=DEV)
    got = []
    for far in (0, 1000, 2 ** 24 + 1, 2 ** 31 - 20):
        a, b = torch.empty_like(q), torch.empty_like(k)
        L.rope(a, q, freqs, offset=far + 13)
        L.rope(b, k, freqs, offset=far)
        got.append(float((a.double() * b.double()).sum()))
    # 16 roundings of 2^-24 relative to |q| |k|, as in _close for either factor
    assert max(got) - min(got) <= 2 * 16 * 2.0 ** -24 * float(q.norm() * k.norm())


def test_gradient_is_the_inverse_and_matches_differences():
    b, t, h, hd, rot = 1, 6, 2, 32, 20
    freqs = L.rope_frequencies(rot, device=DEV)
    x = torch.randn(b, t, h, hd, device=DEV)
    dy = torch.randn(b, t, h, hd, device=DEV)
    dx, y = torch.empty_like(x), torch.empty_like(x)
    L.rope(dx, dy, freqs, offset=3, inverse=True, scale=1.2)
    way = torch.randn_like(x)
    lo, hi = torch.empty_like(x), torch.empty_like(x)
    L.rope(hi, x + 0.5 * way, freqs, offset=3, scale=1.2)
    L.rope(lo, x - 0.5 * way, freqs, offset=3, scale=1.2)
    change, slope = ((hi.double() - lo.double()) * dy.double()).sum(), (dx.double() * way.double()).sum()
    # linear in x: the difference is exact but for fp32 roundings of values of up to a few units
    assert abs(float(change - slope)) <= 32 * 2.0 ** -24 * float((hi.abs() + lo.abs()).double().mul(dy.abs().double()).sum())


def test_another_stream_and_a_captured_call():
    b, t, h, hd = 2, 64, 4, 64
    freqs = L.rope_frequencies(hd, device=DEV)
    x = torch.randn(b, t, h, hd, device=DEV).bfloat16()
    want, y = torch.empty_like(x), torch.zeros_like(x)
    L.rope(want, x, freqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    L.rope(y, x, freqs, stream=side)
    side.synchronize()
    assert torch.equal(y, want)
    y.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.rope(y, x, freqs)
    x.copy_(torch.randn(b, t, h, hd, device=DEV))
    L.rope(want, x, freqs)
    g.replay()
    assert torch.equal(y, want)
    del g
    assert math.isfinite(float(y.float().sum()))
