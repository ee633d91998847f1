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


# --------------------------------------------------------------------------------------------
# finite scores far from zero
# --------------------------------------------------------------------------------------------
def _far_case(dt, sign, e, step, n, m, d, g):
    """Queries and keys whose scores (scale 1) are sign * 32761 * 2^e + step * c_j, c_j whole numbers in [-24, 0], exactly: (181 * 2^x) times
    (181 * 2^y) and a product with a multiple of `step`, all inside every storage type, whose sum f32 holds.  Returns q [n,2,d], k [m,1,d], the
    scores."""
    c = -torch.randint(0, 25, (m,), generator=g)
    top, fine = sign * 32761 * 2.0 ** e, 2.0 ** (round(math.log2(step)) // 2)
    q, k = torch.zeros(n, 2, d), torch.zeros(m, 1, d)
    q[..., 0], k[..., 0] = 181 * 2.0 ** (e // 2), sign * 181 * 2.0 ** (e - e // 2)
    q[..., 1], k[:, 0, 1] = fine, step / fine * c
    scores = top + step * c.double()
    for t in (q, k):
        assert torch.equal(t.to(dt).float(), t)
    assert torch.equal((q[0, 0] * k[:, 0]).sum(-1).double(), scores)
    return q.to(dt), k.to(dt), scores


def _far_expect(got, scores, seen, v, dt, what):
    """The scores are exact, so are their distances from the maximum; a distance times scale log2(e) is rounded twice, and a weight
    whose distance passes 256 is below every other's rounding: 256 * 1.45 * 2^-23 and the exponential's own error stay below 2^-13.  16-bit storage: a
    block may be weighed against a rounded maximum below 2^12, at most 2^-13 of a power of two off.  Twice that, and the usual rest."""
    n, h, d = got.shape
    o, amp = torch.zeros(n, h, d, dtype=torch.float64), torch.zeros(n, h, d, dtype=torch.float64)
    for i in range(n):
        s = scores[seen[i]]
        if s.numel():
            w = torch.softmax(s, 0)
            vv = v.double().cpu()[seen[i], 0]
            o[i], amp[i] = w @ vv, w @ vv.abs()
    tol = _attn_tol(dt, o, amp, scores.numel(), 0, 0.0, _vmax(v)) + 2.0 ** -12 * amp
    _within(got, o, tol, what)


@DT
@pytest.mark.parametrize("sign,e,step", [(1, -5, 0.25), (1, -2, 0.25), (1, 5, 0.25), (-1, 5, 1.0), (1, 10, 4.0), (-1, 15, 256.0), (1, 15, 64.0),
                                         (1, 25, 2.0 ** 16)])
def test_scores_far_from_zero(backend, dt, sign, e, step):
    """Scores of 10^3 to 10^12: a product with scale * log2(e) rounds them by up to thousands of units, their distances from the maximum are
    exact."""
    if dt == F16 and e > 16:
        pytest.skip("no such product of two f16 values")
    top = (sign, e)
    g = torch.Generator().manual_seed(3)
    n, m, d = 40, 330, 32
    q, k, scores = _far_case(dt, sign, e, step, n, m, d, g)
    v = torch.randn(m, 1, d, generator=g).to(dt)
    dq, dk, dv = q.to(backend), k.to(backend), v.to(backend)
    for causal in (False, True):
        out, lse = torch.empty_like(dq), torch.empty(n, 2, device=backend)
        ops.prompt_attention(dq, dk, dv, out, _i32([0, n], backend), _i32([0, m], backend), causal=causal, scale=1.0, lse=lse)
        seen = _seen(n, m, causal)
        _far_expect(out, scores, seen, v, dt, (top, causal))
        want = torch.stack([torch.logsumexp(scores[s], 0) for s in seen])
        assert ((lse.double().cpu() - want[:, None]).abs() <= 2.0 ** -22 * want.abs()[:, None] + 1e-3).all()
    b = 4                                                           # pieces of a prefix and own keys, joined
    out = torch.empty(b, 2, d, dtype=dt, device=backend)
    own_k, own_v = dk[300:].expand(b, 30, 1, d).contiguous(), dv[300:].expand(b, 30, 1, d).contiguous()
    ops.prefix_attention(dq[:b], dk[:300], dv[:300], own_k, own_v, _i32([30, 1, 17, 0], backend), out, scale=1.0)
    seen = torch.arange(m) < 300 + torch.tensor([30, 1, 17, 0])[:, None]
    _far_expect(out, scores, seen, v, dt, (top, "prefix"))


@DT
def test_far_scores_whose_keys_are_shared_by_work_groups(backend, dt):
    g = torch.Generator().manual_seed(4)
    n, m, d = 3, 1500, 32
    assert ops.prompt_splits(1, n, m, 2, 1) > 1
    q, k, scores = _far_case(dt, 1, 14, 64.0, n, m, d, g)
    v = torch.randn(m, 1, d, generator=g).to(dt)
    out = torch.empty(n, 2, d, dtype=dt, device=backend)
    ops.prompt_attention(q.to(backend), k.to(backend), v.to(backend), out, _i32([0, n], backend), _i32([0, m], backend), scale=1.0)
    _far_expect(out, scores, _seen(n, m, True), v, dt, "split")


@DT
def test_random_queries_and_keys_of_large_size(backend, dt):
    """Inputs near the top of f16, 10^6 in the wider types: the softmax of such scores is one key's value unless two meet within rounding."""
    g = torch.Generator().manual_seed(5)
    a, n, m, d = (1.5e4 if dt == F16 else 1e6), 48, 140, 64
    q, k, v = (torch.randn(t, h, d, generator=g) for t, h in ((n, 2), (m, 1), (m, 1)))
    q, k, v = (q * a).clamp(-4 * a, 4 * a).to(dt), (k * a).clamp(-4 * a, 4 * a).to(dt), v.to(dt)
    out = torch.empty(n, 2, d, dtype=dt, device=backend)
    ops.prompt_attention(q.to(backend), k.to(backend), v.to(backend), out, _i32([0, n], backend), _i32([0, m], backend), causal=False)
    s = (q.double()[:, :, None] * k.double()[None, None, :, 0]).sum(-1) * d ** -0.5
    best = s.topk(2, -1)
    slack = (d + 4) * 2.0 ** -24 * (q.double().abs()[:, :, None] * k.double().abs()[None, None, :, 0]).sum(-1).amax(-1) * d ** -0.5
    clear = best.values[..., 0] - best.values[..., 1] > 2 * slack + 100
    assert clear.float().mean() > 0.9
    got = out.float().cpu()
    assert bool(got.isfinite().all()) and got.abs().max() <= v.float().abs().max() * 1.01
    assert torch.equal(out.cpu()[clear], v[:, 0][best.indices[..., 0]][clear])


# --------------------------------------------------------------------------------------------
# offsets that decrease (device data: no host check sees them)
# --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cu_q,cu_k", [
    ([0, 400, 10, 10], [0, 400, 400, 400]),         # one work-group per tile
    ([0, 390, 10, 400], [0, 800, 1600, 2400]),      # shared keys, in this case and those below
    ([10, 0, 400], [0, 1200, 2400]),
    ([0, 200, 150, 400], [0, 2400, 2400, 2400]),
    ([400, 200, 0], [0, 1200, 2400]),
])
@pytest.mark.parametrize("causal", [True, False])
def test_offsets_that_decrease(backend, cu_q, cu_k, causal):
    """Such a call is not specified, but a row is left as it was or holds the result of a sequence that contains it, never what the scratch
    held."""
    g = torch.Generator().manual_seed(6)
    tq, d, m = 400, 32, cu_k[-1]
    q, k, v = (torch.randn(n, 1, d, generator=g) for n in (tq, m, m))
    dq, dk, dv = q.to(backend), k.to(backend), v.to(backend)
    out = torch.full((tq, 1, d), 7.0, device=backend)
    dcu = _i32(cu_q, backend)
    need = ops.prompt_attention_scratch(dq, dk, dcu)
    assert (need > 0) == (m == 2400)
    scratch = torch.full((max(1, need),), math.nan, device=backend)
    ops.prompt_attention(dq, dk, dv, out, dcu, _i32(cu_k, backend), causal=causal, scratch=scratch)
    out = out.cpu()[:, 0]
    fine = (out == 7.0).all(-1)
    for a, b, c, e in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if b > a:
            s = (q[a:b, 0].double() @ k[c:e, 0].double().T * d ** -0.5).masked_fill(~_seen(b - a, e - c, causal), -INF)
            w, vv = torch.nan_to_num(torch.softmax(s, -1)), v[c:e, 0].double()
            smax = (q[a:b, 0].abs() @ k[c:e, 0].abs().T).max().item() * d ** -0.5 if e > c else 0.0
            fine[a:b] |= ((out[a:b].double() - w @ vv).abs() <= _attn_tol(F32, w @ vv, w @ vv.abs(), e - c, d, smax, _vmax(v))).all(-1)
    assert bool(fine.all()), (~fine).nonzero()[:, 0].tolist()


def test_many_sequences_do_not_share_keys(emu_lib):
    """`splits` is a hint: with more sequences than the joining launch can look over the keys of a tile stay with one work-group."""
    g = torch.Generator().manual_seed(7)
    n, d = 5000, 8
    q, k, v = (torch.randn(n, 1, d, generator=g) for _ in range(3))
    cu = torch.arange(n + 1, dtype=torch.int32)
    want, out = torch.empty_like(q), torch.empty_like(q)
    ops.prompt_attention(q, k, v, want, cu)
    scratch = torch.full((n * 2 * (d + 4),), math.nan)
    P = lib.STRUCTS["pp_prompt_attention_params"]()
    P.dtype, P.causal, P.scale, P.splits = lib.CONSTS["PP_F32"], 1, d ** -0.5, 2
    P.q, P.k, P.v, P.out, P.cu_q, P.cu_k = (t.data_ptr() for t in (q, k, v, out, cu, cu))
    P.q_row = P.k_row = P.v_row = P.out_row = d
    P.B, P.Tq, P.Tk, P.H, P.KH, P.D = n, n, n, 1, 1, d
    P.scratch, P.scratch_bytes = scratch.data_ptr(), scratch.numel() * 4
    emu_lib.call("pp_prompt_attention", 0, P)
    assert torch.equal(out, want) and bool(scratch.isnan().all())


# --------------------------------------------------------------------------------------------
# lengths at the end of the accepted range
# --------------------------------------------------------------------------------------------
def _prompt_params(cu_k, tk, t):
    P = lib.STRUCTS["pp_prompt_attention_params"]()
    P.dtype, P.causal, P.scale = lib.CONSTS["PP_F32"], 0, 1.0
    P.q, P.k, P.v, P.out = (x.data_ptr() for x in t[:4])
    P.cu_q, P.cu_k = t[4].data_ptr(), cu_k.data_ptr()
    P.q_row = P.k_row = P.v_row = P.out_row = 8
    P.B, P.Tq, P.Tk, P.H, P.KH, P.D = 1, 1, tk, 1, 1, 8
    return P


def test_lengths_that_a_walk_over_the_keys_cannot_count(emu_lib):
    """Keys are counted in 32 bits, up to three blocks beyond the last: lengths above 2^31 - 1024 are refused.  (No such tensor is made: the
    offsets and lengths of the accepted calls leave one key.)"""
    t = (torch.ones(1, 8), torch.ones(1, 8), torch.full((1, 8), 3.0), torch.zeros(1, 8), torch.tensor([0, 1], dtype=torch.int32))
    cu_k = torch.tensor([0, 1], dtype=torch.int32)
    for tk in (2 ** 31 - 1, 2 ** 31 - 1023):
        with pytest.raises(RuntimeError, match="2\\^31 - 1024"):
            emu_lib.call("pp_prompt_attention", 0, _prompt_params(cu_k, tk, t))
    emu_lib.call("pp_prompt_attention", 0, _prompt_params(cu_k, 2 ** 31 - 1024, t))
    assert bool((t[3] == 3).all())
    scratch, own_len = torch.zeros(4 * 12), torch.ones(1, dtype=torch.int32)
    for p, s in ((2 ** 31 - 1, 0), (2 ** 31 - 1023, 0), (0, 2 ** 31 - 1023), (0, 2 ** 31 - 1024)):
        P = lib.STRUCTS["pp_prefix_attention_params"]()
        P.dtype, P.scale = lib.CONSTS["PP_F32"], 1.0
        P.q, P.kp, P.vp, P.ko, P.vo, P.out = (t[i].data_ptr() for i in (0, 1, 2, 1, 2, 3))
        P.own_len, P.scratch, P.scratch_bytes = own_len.data_ptr(), scratch.data_ptr(), scratch.numel() * 4
        P.kp_row = P.vp_row = P.ko_row = P.vo_row = 8
        P.prefix_splits, P.own_splits = int(p > 0), int(s > 0)
        P.B, P.L, P.P, P.S, P.H, P.KH, P.D = 1, 1, p, s, 1, 1, 8
        if s == 2 ** 31 - 1024:
            t[3].zero_()
            emu_lib.call("pp_prefix_attention", 0, P)
            assert bool((t[3] == 3).all())
        else:
            with pytest.raises(RuntimeError, match="2\\^31 - 1024"):
                emu_lib.call("pp_prefix_attention", 0, P)
