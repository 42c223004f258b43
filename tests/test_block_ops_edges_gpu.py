"""Rotary positions, norms around a block and windowed attention at the edge of what their header allows."""
import pytest

torch = pytest.importorskip("torch")

import llmt_b200 as L

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
