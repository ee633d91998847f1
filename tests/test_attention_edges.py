"""Edges of prompt_attention and prefix_attention: keys whose rows lie closer together than their channels, scores far from zero, offsets that
decrease, lengths at the end of the accepted range.  References and tolerances are those of test_norm_attention."""
import math

import pytest
import torch

from comfyui_propainter_nodes_amd import lib, ops
from test_norm_attention import BF16, DT, F16, F32, U, _attend_ref, _attn_tol, _cu, _seen, _within

INF = math.inf


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _vmax(v):
    return torch.nan_to_num(v.float(), nan=0.0, posinf=0.0, neginf=0.0).abs().max().item()


def _expect(got, q, k, v, seen, what):
    """got against the formula; got, q [n,H,D], k, v [m,KH,D]."""
    dt, d = q.dtype, q.shape[2]
    o, amp, _, smax = _attend_ref(q.double().cpu(), k.double().cpu(), v.double().cpu(), seen, d ** -0.5)
    _within(got, o, _attn_tol(dt, o, torch.nan_to_num(amp, nan=0.0, posinf=0.0), k.shape[0], d, smax, _vmax(v)), what)


# --------------------------------------------------------------------------------------------
# rows of keys and values that lie closer together than their channels
# --------------------------------------------------------------------------------------------
@DT
@pytest.mark.parametrize("bad", [INF, -INF, math.nan])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_one_key_with_a_value_that_is_not_finite(backend, dt, bad, d):
    """One key: its value is the result, an infinity stays an infinity.  (The block's other rows repeat it when the stride of a single row
    counts as 0: 0 x inf.)"""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(3, 4, d, generator=g).to(dt), *(torch.randn(1, 2, d, generator=g).to(dt) for _ in range(2)))
    v[0, 0, 5], v[0, 1, d - 1] = bad, -bad
    dq, dk, dv = q.to(backend), k.to(backend), v.to(backend)
    for causal in (False, True):        # causal: only the last of the three rows sees the key
        out = torch.empty_like(dq)
        ops.prompt_attention(dq, dk, dv, out, _i32([0, 3], backend), _i32([0, 1], backend), causal=causal)
        _expect(out, q, k, v, _seen(3, 1, causal), ("prompt", causal))
    none = torch.empty(0, 2, d, dtype=dt, device=backend)
    out = torch.empty_like(dq)
    ops.prefix_attention(dq, dk, dv, none.expand(3, 0, 2, d), none.expand(3, 0, 2, d), _i32([0, 0, 0], backend), out)
    _expect(out, q, k, v, _seen(3, 1, False), "prefix of one key")
    ops.prefix_attention(dq, none, none, dk.expand(3, 1, 2, d).contiguous(), dv.expand(3, 1, 2, d).contiguous(), _i32([1, 1, 0], backend), out)
    seen = torch.tensor([[True], [True], [False]])
    _expect(out, q, k, v, seen, "one own key")


@DT
@pytest.mark.parametrize("n", [10, 64, 70])
def test_expanded_and_overlapping_rows(backend, dt, n):
    """Keys and values as expanded views (stride 0) and as sliding windows over a line (a stride below the channels)."""
    g = torch.Generator().manual_seed(2)
    d, step, h = 32, 16, 2
    q = torch.randn(5, h, d, generator=g).to(dt)
    line = torch.randn(2, n * step + d, generator=g).to(dt)
    line[1, (n - 1) * step + 20] = INF      # channel 20 of the last row; it would be channel 4 of a row behind it
    line = line.to(backend)
    k, v = (line[i].as_strided((n, 1, d), (step, d, 1)) for i in range(2))
    one = torch.randn(2, 1, 1, d, generator=g).to(dt)
    one[1, 0, 0, 7] = -INF
    one = one.to(backend)
    dq = q.to(backend)
    for name, kk, vv in (("windows", k, v), ("expanded", one[0].expand(n, 1, d), one[1].expand(n, 1, d))):
        for causal in (False, True):
            out = torch.empty_like(dq)
            ops.prompt_attention(dq, kk, vv, out, _i32([0, 5], backend), _i32([0, n], backend), causal=causal)
            _expect(out, q, kk.cpu(), vv.cpu(), _seen(5, n, causal), (name, causal))
        out = torch.empty_like(dq)
        none = kk[:0].expand(0, 1, d)
        ops.prefix_attention(dq, kk, vv, none.expand(5, 0, 1, d), none.expand(5, 0, 1, d), _i32([0] * 5, backend), out)
        _expect(out, q, kk.cpu(), vv.cpu(), _seen(5, n, False), (name, "prefix"))
