"""Group norm with an activation, attention over packed sequences and attention behind a shared prefix against their formulas in 64
bits, on the emulator and on the MI355X.

Tolerances are bounds, element by element, from the formulas and the storage types; u = eps / 2 is the largest relative rounding error.
  group norm: the sums are doubles, so the f32 steps count: two subtractions, the factor (1/std and gamma rounded, their product, the product
    with it), the sum with beta: 6 roundings of at most |n gamma| + |beta| each; an activation has a slope below 1.13 and is within 8 roundings of
    its value; together below 16 * 2^-24 * (|n gamma| + |beta|).  Then the skip's sum and the rounding to storage.
  attention, with w = softmax weights, A = sum_j w_j |v_j| (what relative errors of the weights can move the result by), S = the largest
    scale * sum_d |q_d k_d| of the case:
    scores: D products summed in f32, at most (D + 4) 2^-24 S off, argument of exp2 rounded once (2^-24 of at most 2 S), so each weight is at most
    (D + 8) S 2^-23 off, and the sums over n keys and the rescales at most (n + 16) 2^-23;
    16-bit storage: each probability is rounded once more (u; f16 below 2^-14: 2^-25 absolute, against a sum of at least 1), and so is the result.
"""
import math

import pytest
import torch
import torch.nn.functional as F

from comfyui_propainter_nodes_amd import lib, ops

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
DT = pytest.mark.parametrize("dt", [F16, BF16, F32], ids=["f16", "bf16", "f32"])
gpu_only = pytest.mark.gpu


def _within(got, ref, tol, what=""):
    got, ref, tol = got.double().cpu(), ref.double().cpu(), tol.double().cpu()
    assert torch.equal(got.isnan(), ref.isnan()), what
    inf = ref.isinf()
    assert torch.equal(got[inf], ref[inf]), what
    fine = ref.isfinite()
    over = ((got - ref).abs() - tol)[fine]
    assert over.numel() == 0 or over.max().item() <= 0, (what, over.max().item(), tol[fine].max().item())


# --------------------------------------------------------------------------------------------
# group norm
# --------------------------------------------------------------------------------------------
ACTS = {"none": lambda t: t, None: lambda t: t, "relu": F.relu, "leaky": lambda t: F.leaky_relu(t, 0.1), "sigmoid": torch.sigmoid,
        "tanh": torch.tanh, "gelu": F.gelu, "silu": F.silu}


def _groupnorm_ref(x, groups, gamma, beta, act, skip, relu_post, eps):
    x = x.double().cpu()
    n, h, w, c = x.shape
    v = x.reshape(n, h * w, groups, c // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((v - mean) / (var + eps).sqrt()).reshape(n, h, w, c)
    g = gamma.double().cpu() if gamma is not None else torch.ones(c, dtype=torch.float64)
    b = beta.double().cpu() if beta is not None else torch.zeros(c, dtype=torch.float64)
    y = ACTS[act](z * g + b)
    tol = 16 * 2.0 ** -24 * ((z * g).abs() + b.abs())
    if skip is not None:
        y = y + skip.double().cpu()
        tol = tol + 2.0 ** -23 * y.abs()
    return (F.relu(y) if relu_post else y), tol


def _groupnorm_case(dev, dt, shape, groups, act, skip=False, affine=True, pitch=0, inplace=False, eps=1e-5, mean=0.0, seed=1):
    g = torch.Generator().manual_seed(seed)
    n, h, w, c = shape
    def view():
        return torch.full((n, h, w, c + pitch), 7.0, dtype=dt, device=dev)[..., :c]
    x = view()
    x.copy_((torch.randn(shape, generator=g) * (0.5 + torch.rand(c, generator=g)) + torch.randn(c, generator=g) + mean).to(dt))
    gamma = (1 + 0.2 * torch.randn(c, generator=g)).to(dev) if affine else None
    beta = (0.2 * torch.randn(c, generator=g)).to(dev) if affine else None
    sk = torch.randn(shape, generator=g).to(dt).to(dev) if skip else None
    ref, tol = _groupnorm_ref(x, groups, gamma, beta, act, sk, skip, eps)
    y = x if inplace else view()
    got = ops.groupnorm(x, y, groups, gamma, beta, act=act, act_param=0.1, skip=sk, relu_post=skip, eps=eps)
    assert got is y
    _within(got, ref, tol + U[dt] * ref.abs() + (2.0 ** -25 if dt == F16 else 0.0), (dt, shape, groups, act))
    if pitch:
        assert bool((y._base[..., c:] == 7).all())   # the channels beside the view


@DT
@pytest.mark.parametrize("shape,groups,act,kw", [
    ((2, 9, 7, 64), 8, "relu", dict()),
    ((1, 1, 1, 32), 4, "none", dict()),
    ((1, 5, 1, 8), 1, "silu", dict()),
    ((3, 6, 5, 320), 32, "gelu", dict()),                      # groups of 10: a 16-byte vector straddles groups
    ((2, 4, 3, 33), 11, "sigmoid", dict()),                    # odd channels: single elements
    ((2, 4, 3, 33), 1, "tanh", dict(affine=False)),
    ((1, 3, 5, 24), 24, "leaky", dict()),                      # one channel per group
    ((2, 7, 6, 48), 6, "relu", dict(skip=True)),
    ((2, 7, 6, 40), 4, "silu", dict(pitch=24, inplace=True)),
    ((2, 7, 6, 40), 4, "silu", dict(pitch=3)),                 # a pitch that breaks the 16-byte alignment
    ((1, 3, 3, 2304), 2, "none", dict()),                      # more columns than a work-group holds at once
    ((1, 2, 3, 515), 5, "none", dict()),
    ((4, 40, 33, 64), 8, "relu", dict()),                      # several pieces per image
    ((1, 32, 32, 16), 2, "silu", dict(skip=True)),             # 1024 vectors a group in 16-bit storage: the largest held in registers
    ((1, 32, 33, 16), 2, "silu", dict(skip=True)),             # ... and the next, in two launches
])
def test_groupnorm(backend, dt, shape, groups, act, kw):
    _groupnorm_case(backend, dt, shape, groups, act, **kw)


def test_groupnorm_of_data_far_from_zero(backend):
    """mean / std = 10^4: sums of squares in f32 would leave no digit of the variance."""
    _groupnorm_case(backend, F32, (2, 24, 16, 32), 4, "none", mean=1e4)
    _groupnorm_case(backend, F32, (1, 4, 4, 8), 2, "none", mean=3e4, eps=0.0)


@DT
def test_groupnorm_nan_stays_in_its_group(backend, dt):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 6, 5, 64, generator=g).to(dt)
    clean = torch.empty_like(x).to(backend)
    ops.groupnorm(x.to(backend), clean, 8, act="relu")
    x[0, 2, 3, 17] = float("nan")
    x[1, 0, 0, 40] = float("inf")
    y = torch.empty_like(x).to(backend)
    ops.groupnorm(x.to(backend), y, 8, act="relu")
    y, clean = y.float().cpu(), clean.float().cpu()
    bad = torch.zeros(2, 64, dtype=torch.bool)
    bad[0, 16:24] = bad[1, 40:48] = True
    for n in range(2):
        assert bool(y[n][..., bad[n]].isnan().all())
        assert torch.equal(y[n][..., ~bad[n]], clean[n][..., ~bad[n]])


def test_groupnorm_refusals(emu_lib):
    x = torch.zeros(1, 4, 4, 16)
    y = torch.empty_like(x)
    with pytest.raises(ValueError, match="groups"):
        ops.groupnorm(x, y, 3)
    with pytest.raises(ValueError, match="groups"):
        ops.groupnorm(x, y, 0)
    with pytest.raises(ValueError, match="activation"):
        ops.groupnorm(x, y, 4, act="swish")
    with pytest.raises(ValueError, match="shape"):
        ops.groupnorm(x, y[:, :2], 4)
    with pytest.raises(TypeError, match="share a dtype"):
        ops.groupnorm(x, y.half(), 4)
    with pytest.raises(TypeError, match="unsupported dtype"):
        ops.groupnorm(x.double(), y.double(), 4)
    with pytest.raises(ValueError, match="gamma"):
        ops.groupnorm(x, y, 4, torch.ones(8))
    with pytest.raises(ValueError, match="scratch"):
        ops.groupnorm(x, y, 4, scratch=torch.empty(3, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="eps"):
        ops.groupnorm(x, y, 4, eps=-1.0)
    with pytest.raises(KeyError):       # the convolutions do not take the new activation
        ops.conv2d(ops.make_conv_spec(torch.zeros(32, 32, 1, 1), None, F32), [torch.zeros(1, 4, 4, 32)], torch.empty(1, 4, 4, 32), act="silu")
    P = ops._conv2d_params(ops.make_conv_spec(torch.zeros(32, 32, 1, 1), None, F32), [torch.zeros(1, 4, 4, 32)], torch.empty(1, 4, 4, 32))
    P.act = lib.CONSTS["PP_ACT_SILU"]
    with pytest.raises(RuntimeError, match="PP_ACT_SILU"):
        lib.current().call("pp_conv2d", 0, P)
    e = torch.empty(0, 4, 4, 16)
    assert ops.groupnorm(e, torch.empty_like(e), 4).shape == e.shape


# --------------------------------------------------------------------------------------------
# attention: the formula
# --------------------------------------------------------------------------------------------
def _attend_ref(q, k, v, seen, scale):
    """q [n,H,D], k, v [m,KH,D] (64 bits), seen [n,m] -> out, tolerance factor A, lse; a row that sees nothing: 0, -inf.  What a row does
    not see is taken out before any arithmetic."""
    n, h, d = q.shape
    m, kh, _ = k.shape
    out, amp = torch.zeros(n, h, d, dtype=torch.float64), torch.zeros(n, h, d, dtype=torch.float64)
    lse, smax = torch.full((n, h), -math.inf, dtype=torch.float64), 0.0
    for i in range(n):
        js = seen[i].nonzero()[:, 0]
        if js.numel() == 0:
            continue
        kk, vv = k[js].repeat_interleave(h // kh, 1), v[js].repeat_interleave(h // kh, 1)
        s = (q[i][None] * kk).sum(-1) * scale
        w = torch.softmax(s, 0)
        out[i] = (w[..., None] * vv).sum(0)
        amp[i] = (w[..., None] * vv.abs()).sum(0)
        lse[i] = torch.logsumexp(s, 0)
        smax = max(smax, torch.nan_to_num((q[i][None] * kk).abs().sum(-1) * scale, nan=0.0, posinf=0.0).max().item())
    return out, amp, lse, smax


def _attn_tol(dt, out, amp, n, d, smax, vmax):
    f32 = (n + 16 + 2 * (d + 8) * smax) * 2.0 ** -23
    tol = U[dt] * out.abs() + f32 * amp
    if dt != F32:
        tol = tol + U[dt] * amp * (1 + f32)
    if dt == F16:
        tol = tol + n * 2.0 ** -25 * vmax + 2.0 ** -25
    return tol


def _seen(n, m, causal):
    seen = torch.ones(n, m, dtype=torch.bool)
    return seen.tril(m - n) if causal else seen


def _cu(lens, dev):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)) if lens else [0], dtype=torch.int32, device=dev)


def _prompt_ref(q, k, v, lq, lk, causal, scale):
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    outs, tols, lses, a, c = [], [], [], 0, 0
    for n, m in zip(lq, lk):
        o, amp, lse, smax = _attend_ref(q[a:a + n], k[c:c + m], v[c:c + m], _seen(n, m, causal), scale)
        outs.append((o, amp, m, smax))
        lses.append(lse)
        a, c = a + n, c + m
    return outs, lses


def _check_prompt(dev, dt, h, kh, d, lq, lk, causal, layout="plain", scale=None, tail=0, seed=5):
    g = torch.Generator().manual_seed(seed)
    tq, tk = sum(lq) + tail, sum(lk) + tail
    if layout == "fused":       # slices of one projection's output
        assert tq == tk
        qkv = torch.randn(tq, h + 2 * kh, d, generator=g).to(dt).to(dev)
        q, k, v = qkv[:, :h], qkv[:, h:h + kh], qkv[:, h + kh:]
    else:
        q, k, v = (torch.randn(t, n, d, generator=g).to(dt).to(dev) for t, n in ((tq, h), (tk, kh), (tk, kh)))
    if layout == "heads_first":
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    out = torch.full((tq, h, d), 7.0, dtype=dt, device=dev)
    lse = torch.full((tq, h), 7.0, device=dev)
    got = ops.prompt_attention(q, k, v, out, _cu(lq, dev), None if lq is lk else _cu(lk, dev), causal=causal, scale=scale, lse=lse)
    assert got is out
    sc = d ** -0.5 if scale is None else scale
    refs, lses = _prompt_ref(q, k, v, lq, lk, causal, sc)
    vmax, a = v.float().abs().max().item() if tk else 0.0, 0
    for (o, amp, m, smax), ls in zip(refs, lses):
        n = o.shape[0]
        _within(out[a:a + n], o, _attn_tol(dt, o, amp, m, d, smax, vmax), (dt, h, kh, d, lq, lk, causal))
        t = torch.nan_to_num((2 * (d + 8) * smax + m + 16) * 2.0 ** -23 + 2.0 ** -22 * ls.abs(), posinf=0.0)
        _within(lse[a:a + n], ls, t, "lse")
        a += n
    assert bool((out[a:] == 7).all()) and bool((lse[a:] == 7).all())     # rows behind the last sequence


@DT
@pytest.mark.parametrize("h,kh,d,lq,lk,causal,layout", [
    (2, 1, 64, [1], None, True, "plain"),
    (4, 2, 64, [7, 1, 19], None, True, "fused"),
    (3, 3, 32, [5, 0, 33, 2], None, True, "plain"),
    (6, 2, 96, [3, 40], [9, 70], True, "heads_first"),         # queries behind earlier keys
    (2, 2, 128, [45, 45], None, False, "fused"),
    (4, 1, 80, [66], None, True, "plain"),
    (2, 1, 256, [37], None, True, "plain"),
    (1, 1, 8, [6, 4], [2, 0], True, "plain"),                  # fewer keys than queries: rows that see nothing
    (2, 1, 64, [3, 2], [0, 5], False, "plain"),
    (8, 1, 64, [65, 64, 63], None, True, "plain"),
    (5, 5, 40, [130], None, True, "plain"),
])
def test_prompt_attention(backend, dt, h, kh, d, lq, lk, causal, layout):
    _check_prompt(backend, dt, h, kh, d, lq, lq if lk is None else lk, causal, layout)


@DT
@pytest.mark.parametrize("d", [4, 12, 24, 48, 72, 112, 160, 200, 248])
def test_prompt_attention_head_sizes(backend, dt, d):
    if dt != F32 and d % 8:
        pytest.skip("16-byte rows")
    _check_prompt(backend, dt, 2, 1, d, [11, 34], [20, 34], True)


@DT
def test_prompt_attention_scales_and_tail_rows(backend, dt):
    _check_prompt(backend, dt, 2, 1, 32, [9, 21], [9, 21], True, scale=1.0, tail=5)
    _check_prompt(backend, dt, 2, 2, 32, [40], [40], True, scale=1e-6)
    _check_prompt(backend, dt, 2, 1, 32, [], [], True, tail=3)


@DT
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prompt_attention_unseen_values_never_reach_a_row(backend, dt, bad):
    """Tokens of other sequences, of the future and behind the last sequence hold NaN / infinities."""
    g = torch.Generator().manual_seed(9)
    lens, h, kh, d = [40, 7, 70], 4, 2, 64
    t = sum(lens) + 9
    q, k, v = (torch.randn(t, n, d, generator=g).to(dt) for n in (h, kh, kh))
    want = torch.empty(t, h, d, dtype=dt, device=backend)
    ops.prompt_attention(q.to(backend), k.to(backend), v.to(backend), want, _cu(lens, backend))
    k2, v2 = k.clone(), v.clone()
    first_bad = [20, 47, 100]        # a token of each sequence (its own later rows see it), and everything behind the last
    for r in (*first_bad[:1], first_bad[2]):
        k2[r, 0] = bad
        v2[r, :, 5] = bad
    k2[40:47] = bad                  # the whole second sequence
    v2[40:47] = bad
    k2[sum(lens):] = bad
    v2[sum(lens):] = bad
    got = torch.empty_like(want)
    ops.prompt_attention(q.to(backend), k2.to(backend), v2.to(backend), got, _cu(lens, backend))
    want, got = want.float().cpu(), got.float().cpu()
    tol = 4 * U[dt] * v.float().abs().max()      # (a guarded sub-tile multiplies the same operands; other rescale points are allowed)
    for a, b in ((0, 20), (47, 100)):
        assert (want[a:b] - got[a:b]).abs().max() <= tol, (a, b)
    assert bool(got[100:117, 2:, 5].isfinite().logical_not().all())     # rows that do see it (head group 1: only its V is bad)
    assert (want[100:117, 2:, 6:] - got[100:117, 2:, 6:]).abs().max() <= tol
    if math.isinf(bad):
        assert bool((got[100:117, 2:, 5] == bad).all())


def test_prompt_attention_offsets_out_of_range_stay_inside(emu_lib):
    """Offsets are device data: values out of range are clamped, negative lengths are empty; nothing outside the tensors is touched."""
    q, k, v = torch.randn(20, 2, 32), torch.randn(12, 1, 32), torch.randn(12, 1, 32)
    for cu_q, cu_k in (([-5, 9, 2000], [0, 5, 900]), ([0, 15, 8, 20], [12, 3, -4, 12]), ([30, 30], [0, 12]), ([0, 20], [2**31 - 1, -2**31])):
        out = torch.full((20, 2, 32), 7.0)
        ops.prompt_attention(q, k, v, out, torch.tensor(cu_q, dtype=torch.int32), torch.tensor(cu_k, dtype=torch.int32))
        assert bool(out.isfinite().all())


@DT
@pytest.mark.parametrize("lq,lk,causal", [([3, 1], [1100, 900], True), ([40], [800], False), ([800], [800], True), ([2, 0, 5], [3, 2400, 0], True)])
def test_prompt_attention_keys_shared_by_work_groups(backend, dt, lq, lk, causal):
    """Few rows with many keys: the keys of a tile go to several work-groups; parts without a key, rows without one, rows behind the last
    sequence (tail of q / k / v beyond every offset)."""
    assert ops.prompt_splits(len(lq), sum(lq) + 4, sum(lk) + 4, 2, 1) > 1
    _check_prompt(backend, dt, 2, 1, 32, lq, lk, causal, tail=4)


def test_attention_in_place(backend):
    g = torch.Generator().manual_seed(71)
    q, k, v = (torch.randn(70, n, 64, generator=g).to(F16).to(backend) for n in (4, 2, 2))
    cu, want = _cu([30, 40], backend), torch.empty_like(q)
    ops.prompt_attention(q, k, v, want, cu)
    x = q.clone()
    ops.prompt_attention(x, k, v, x, cu)
    assert torch.equal(x, want)
    n = torch.tensor([3, 0], dtype=torch.int32, device=backend)
    own = torch.randn(2, 3, 2, 64, generator=g).to(F16).to(backend)
    ops.prefix_attention(q[:2], k, v, own, own, n, want[:2])
    x = q[:2].clone()
    ops.prefix_attention(x, k, v, own, own, n, x)
    assert torch.equal(x, want[:2])
    wide = torch.zeros(70, 2, 160, device=backend)
    with pytest.raises(RuntimeError, match="cannot be q"):
        ops.prompt_attention(wide, wide, wide, wide, cu)


def test_prompt_attention_split_scratch(emu_lib):
    q, k = torch.zeros(2, 2, 32), torch.zeros(1024, 1, 32)
    cu_q, cu_k, out = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([0, 1024], dtype=torch.int32), torch.empty(2, 2, 32)
    need = ops.prompt_attention_scratch(q, k, cu_q)
    assert need == 2 * 2 * 4 * 36
    ops.prompt_attention(q, k, k, out, cu_q, cu_k, scratch=torch.empty(need))
    with pytest.raises(ValueError, match="scratch"):
        ops.prompt_attention(q, k, k, out, cu_q, cu_k, scratch=torch.empty(need - 1))


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_attention_more_tiles_than_fit_at_once(backend, causal):
    """More tiles than the chip holds at once, several sequences, spare tile numbers between them: every row comes out once."""
    lq, lk = [30, 0, 1, 17, 40, 8], [30, 5, 40, 9, 40, 0]
    h = kh = 100
    assert (sum(lq) // 128 + len(lq)) * kh > 512
    _check_prompt(backend, F16, h, kh, 32, lq, lk, causal, tail=2)


@gpu_only
def test_prompt_attention_many_long_tiles(hip_lib):
    _check_prompt(torch.device("cuda:0"), BF16, 64, 8, 64, [300, 900, 1, 512, 0, 77], [300, 1000, 700, 512, 3, 77], True)


def test_prompt_attention_many_sequences(backend):
    """The search over the offsets takes more than one step beyond 64 sequences."""
    lens = [(7 * i) % 5 for i in range(150)]
    _check_prompt(backend, F16, 2, 1, 32, lens, lens, True, tail=2)


def test_prompt_attention_refusals(emu_lib):
    q, k = torch.zeros(6, 4, 64), torch.zeros(6, 2, 64)
    out, cu = torch.empty_like(q), torch.tensor([0, 6], dtype=torch.int32)
    with pytest.raises(ValueError, match="shapes"):
        ops.prompt_attention(q, torch.zeros(6, 3, 64), torch.zeros(6, 3, 64), out, cu)
    with pytest.raises(ValueError, match="shapes"):
        ops.prompt_attention(q, k, k[:, :, :32], out, cu)
    with pytest.raises(ValueError, match="last dim"):
        ops.prompt_attention(q, k.transpose(1, 2).contiguous().transpose(1, 2), k, out, cu)
    with pytest.raises(ValueError, match="int32"):
        ops.prompt_attention(q, k, k, out, cu.long())
    with pytest.raises(ValueError, match="int32"):
        ops.prompt_attention(q, k, k, out, cu, torch.tensor([0, 3, 6], dtype=torch.int32))
    with pytest.raises(TypeError, match="share a dtype"):
        ops.prompt_attention(q, k.half(), k.half(), out, cu)
    with pytest.raises(ValueError, match="expanded"):
        ops.prompt_attention(q, k, k, torch.empty(1, 4, 64).expand(6, 4, 64), cu)
    with pytest.raises(ValueError, match="lse"):
        ops.prompt_attention(q, k, k, out, cu, lse=torch.empty(6, 2))
    with pytest.raises(RuntimeError, match="scale"):
        ops.prompt_attention(q, k, k, out, cu, scale=-1.0)
    with pytest.raises(RuntimeError, match="scale"):
        ops.prompt_attention(q, k, k, out, cu, scale=math.inf)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ops.prompt_attention(*(torch.zeros(6, 2, 20, dtype=F16) for _ in range(4)), cu)
    with pytest.raises(RuntimeError, match="up to 256"):
        ops.prompt_attention(*(torch.zeros(6, 2, 264, dtype=F16) for _ in range(4)), cu)
    odd = torch.zeros(6, 2, 65)[:, :, :64]
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.prompt_attention(q, odd, odd, out, cu)
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.prompt_attention(q, torch.zeros(6 * 2 * 64 + 1)[1:].view(6, 2, 64), k, out, cu)


# --------------------------------------------------------------------------------------------
# attention behind a shared prefix
# --------------------------------------------------------------------------------------------
def _check_prefix(dev, dt, h, kh, d, b, new, p, s, lens, layout="plain", seed=6, three=False):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, new, h, d, generator=g).to(dt).to(dev)
    kp, vp = (torch.randn(p, kh, d, generator=g).to(dt).to(dev) for _ in range(2))
    ko, vo = (torch.randn(b, s, kh, d, generator=g).to(dt).to(dev) for _ in range(2))
    for i, n in enumerate(lens):        # what lies behind a sequence's own keys
        ko[i, max(0, n):] = math.nan
        vo[i, max(0, n):] = math.nan
    if layout == "heads_first":
        q, ko, vo = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, ko, vo))
        kp, vp = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (kp, vp))
    own = torch.tensor(lens, dtype=torch.int32, device=dev)
    out = torch.full((b, new, h, d), 7.0, dtype=dt, device=dev)
    if three:
        got = ops.prefix_attention(q[:, 0], kp, vp, ko, vo, own, out[:, 0])
        assert got.shape == (b, h, d)
    else:
        assert ops.prefix_attention(q, kp, vp, ko, vo, own, out) is out
    vmax = max(vp.float().abs().max().item() if p else 0.0, torch.nan_to_num(vo.float()).abs().max().item() if s else 0.0)
    for i, n in enumerate(lens):
        n = max(0, min(n, s))
        kk, vv = torch.cat([kp, ko[i, :n]]).double().cpu(), torch.cat([vp, vo[i, :n]]).double().cpu()
        seen = torch.zeros(new, p + n, dtype=torch.bool)
        for t in range(new):
            seen[t, :p + max(0, n - new + t + 1)] = True
        o, amp, _, smax = _attend_ref(q[i].double().cpu(), kk, vv, seen, d ** -0.5)
        _within(out[i], o, _attn_tol(dt, o, amp, p + n, d, smax, vmax), (dt, h, kh, d, b, new, p, s, lens, i))


@DT
@pytest.mark.parametrize("h,kh,d,b,new,p,s,lens,kw", [
    (2, 1, 64, 2, 1, 70, 17, [17, 3], dict(three=True)),
    (8, 2, 64, 3, 1, 300, 9, [1, 9, 5], dict()),
    (4, 2, 96, 2, 3, 33, 20, [3, 20], dict(layout="heads_first")),
    (3, 3, 32, 2, 2, 1, 5, [2, 1], dict()),                    # a sequence whose first new token has only the prefix
    (2, 1, 128, 2, 1, 0, 40, [40, 0], dict()),                 # no prefix; a row without any key
    (2, 2, 80, 2, 1, 50, 0, [0, 0], dict()),                   # no own keys
    (2, 1, 32, 2, 3, 0, 6, [1, -4], dict()),
    (2, 1, 32, 1, 1, 0, 0, [0], dict()),
    (40, 1, 32, 2, 4, 65, 7, [7, 99], dict()),                 # 160 rows per sequence: two tiles; a length past the cache
    (1, 1, 256, 2, 1, 40, 3, [3, 2], dict()),
])
def test_prefix_attention(backend, dt, h, kh, d, b, new, p, s, lens, kw):
    _check_prefix(backend, dt, h, kh, d, b, new, p, s, lens, **kw)


def test_prefix_attention_splits_agree(backend):
    """Long ranges are cut into pieces that are joined again."""
    _check_prefix(backend, F16, 2, 1, 32, 3, 1, 1500, 600, [600, 1, 257])


def test_prefix_attention_refusals(emu_lib):
    q, kp, ko = torch.zeros(2, 1, 4, 64), torch.zeros(9, 2, 64), torch.zeros(2, 5, 2, 64)
    out, own = torch.empty_like(q), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="shapes"):
        ops.prefix_attention(q, kp, kp, ko[:1], ko[:1], own, out)
    with pytest.raises(ValueError, match="shapes"):
        ops.prefix_attention(q, kp[:, :, :32], kp, ko, ko, own, out)
    with pytest.raises(ValueError, match="own_len"):
        ops.prefix_attention(q, kp, kp, ko, ko, own.long(), out)
    with pytest.raises(TypeError, match="share a dtype"):
        ops.prefix_attention(q, kp.half(), kp.half(), ko, ko, own, out)
    with pytest.raises(ValueError, match="expanded"):
        ops.prefix_attention(q, kp, kp, ko, ko, own, torch.empty(1, 1, 4, 64).expand(2, 1, 4, 64))
    with pytest.raises(ValueError, match="scratch"):
        ops.prefix_attention(q, kp, kp, ko, ko, own, out, scratch=torch.empty(10))
    with pytest.raises(RuntimeError, match="scale"):
        ops.prefix_attention(q, kp, kp, ko, ko, own, out, scale=0.0)
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.prefix_attention(q, torch.zeros(9, 2, 65)[:, :, :64], kp, ko, ko, own, out)
    P = lib.STRUCTS["pp_prefix_attention_params"]()
    with pytest.raises(RuntimeError, match="null"):
        lib.current().call("pp_prefix_attention", 0, P)


def test_sizes_that_no_launch_holds(emu_lib):
    """Sizes whose products leave 64 bits are refused before anything is computed from them."""
    one = torch.zeros(64)
    at = one.data_ptr()
    P = lib.STRUCTS["pp_prefix_attention_params"]()
    P.q = P.kp = P.vp = P.ko = P.vo = P.own_len = P.out = P.scratch = at
    P.prefix_splits = P.own_splits = 1
    P.scale, P.B, P.L, P.H, P.KH, P.D, P.P, P.S = 1.0, 1 << 24, 1 << 20, 1 << 20, 1 << 20, 8, 1, 1
    with pytest.raises(RuntimeError, match="2\\^24 rows"):
        emu_lib.call("pp_prefix_attention", 0, P)
    P = lib.STRUCTS["pp_prompt_attention_params"]()
    P.q = P.k = P.v = P.out = P.cu_q = P.cu_k = at
    P.scale, P.B, P.Tq, P.Tk, P.H, P.KH, P.D = 1.0, 1 << 29, 1 << 30, 1, 1 << 20, 1 << 20, 8
    with pytest.raises(RuntimeError, match="too large"):
        emu_lib.call("pp_prompt_attention", 0, P)
    P.B, P.Tq, P.H, P.KH = 1, 1 << 30, 64, 64
    with pytest.raises(RuntimeError, match="2\\^32 threads"):
        emu_lib.call("pp_prompt_attention", 0, P)
    P = lib.STRUCTS["pp_groupnorm_params"]()
    P.x = P.y = P.partials = at
    P.N, P.HW, P.C, P.groups, P.x_ldc, P.y_ldc, P.nchunks = 1, 1 << 50, 8, 1, 8, 8, 1
    with pytest.raises(RuntimeError, match="HW"):
        emu_lib.call("pp_groupnorm", 0, P)


# --------------------------------------------------------------------------------------------
# together
# --------------------------------------------------------------------------------------------
def test_map_to_prompt_to_continuation(backend):
    """A block over a channels-last map: group norm + SiLU, q | k | v by a 1x1 convolution, attention of its tokens, then a batch of
    continuations that share those tokens as their prefix -- each step against its formula, and the continuation's first token against one long prompt."""
    dev, g = backend, torch.Generator().manual_seed(11)
    h, kh, d, b = 4, 2, 32, 3
    c, width = 64, (h + 2 * kh) * d
    x = torch.randn(1, 6, 7, c, generator=g).to(F16).to(dev)
    gamma, beta = 1 + 0.1 * torch.randn(c, generator=g), 0.1 * torch.randn(c, generator=g)
    z = torch.empty_like(x)
    ops.groupnorm(x, z, 8, gamma.to(dev), beta.to(dev), act="silu")
    ref, tol = _groupnorm_ref(x, 8, gamma, beta, "silu", None, False, 1e-5)
    _within(z, ref, tol + U[F16] * ref.abs() + 2.0 ** -25)
    spec = ops.make_conv_spec(torch.randn(width, c, 1, 1, generator=g) * c ** -0.5, None, F16).to(dev)
    qkv = torch.empty(1, 6, 7, width, dtype=F16, device=dev)
    ops.conv2d(spec, [z], qkv)
    t = qkv.view(42, h + 2 * kh, d)
    q, k, v = t[:, :h], t[:, h:h + kh], t[:, h + kh:]
    out = torch.empty(42, h, d, dtype=F16, device=dev)
    ops.prompt_attention(q, k, v, out, _cu([42], dev))
    o, amp, _, smax = _attend_ref(q.double().cpu(), k.double().cpu(), v.double().cpu(), _seen(42, 42, True), d ** -0.5)
    _within(out, o, _attn_tol(F16, o, amp, 42, d, smax, v.abs().max().item()))
    new = torch.randn(b, h + 2 * kh, d, generator=g).to(F16).to(dev)
    own_k, own_v = torch.zeros(b, 4, kh, d, dtype=F16, device=dev), torch.zeros(b, 4, kh, d, dtype=F16, device=dev)
    own_k[:, 0], own_v[:, 0] = new[:, h:h + kh], new[:, h + kh:]
    step = torch.empty(b, h, d, dtype=F16, device=dev)
    ops.prefix_attention(new[:, :h], k, v, own_k, own_v, torch.ones(b, dtype=torch.int32, device=dev), step)
    for i in range(b):          # the same token as the 43rd of one prompt
        all_k, all_v = torch.cat([k, new[i:i + 1, h:h + kh]]), torch.cat([v, new[i:i + 1, h + kh:]])
        one = torch.empty(1, h, d, dtype=F16, device=dev)
        ops.prompt_attention(new[i:i + 1, :h], all_k, all_v, one, _cu([1], dev), _cu([43], dev))
        o, amp, _, smax = _attend_ref(new[i:i + 1, :h].double().cpu(), all_k.double().cpu(), all_v.double().cpu(), _seen(1, 43, True), d ** -0.5)
        tol = _attn_tol(F16, o, amp, 43, d, smax, all_v.abs().max().item())
        _within(step[i:i + 1], o, tol)
        _within(one, o, tol)


# --------------------------------------------------------------------------------------------
# the encoder that calls it
# --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hw", [(40, 56)])
def test_raft_encoder_with_group_norm(backend, hw):
    """BasicEncoder(norm_fn="group"): 8 groups in the stem, planes // 8 in the blocks, against torch on the same weights.  The 16
    convolutions run as two-term f16 splits (2^-20 of each operand) over at most 1152 products, the norms bring every map back to about
    unit size, and nothing amplifies: 16 layers of 1152^0.5 * 2^-19 stay below 2e-3 of the largest output."""
    from comfyui_propainter_nodes_amd import raft

    g = torch.Generator().manual_seed(21)
    p = {}

    def conv(name, co, ci, k):
        p[name + ".weight"] = torch.randn(co, ci, k, k, generator=g) * (ci * k * k) ** -0.5
        p[name + ".bias"] = 0.1 * torch.randn(co, generator=g)

    def affine(name, c):
        p[name + ".weight"], p[name + ".bias"] = 1 + 0.2 * torch.randn(c, generator=g), 0.2 * torch.randn(c, generator=g)

    conv("conv1", 64, 3, 7)
    affine("norm1", 64)
    ci = 64
    for layer, dim, stride in (("layer1", 64, 1), ("layer2", 96, 2), ("layer3", 128, 2)):
        for i, st in ((0, stride), (1, 1)):
            pre = f"{layer}.{i}."
            conv(pre + "conv1", dim, ci, 3)
            conv(pre + "conv2", dim, dim, 3)
            affine(pre + "norm1", dim)
            affine(pre + "norm2", dim)
            if st != 1:
                conv(pre + "downsample.0", dim, ci, 1)
                affine(pre + "norm3", dim)
            ci = dim
    conv("conv2", 256, 128, 1)
    frames = torch.rand(2, *hw, 3, generator=g) * 2 - 1

    def norm(x, name):
        return F.group_norm(x, x.shape[1] // 8, p[name + ".weight"].double(), p[name + ".bias"].double(), 1e-5)

    def cv(x, name, **kw):
        return F.conv2d(x, p[name + ".weight"].double(), p[name + ".bias"].double(), **kw)

    x = F.relu(norm(cv(frames.double().permute(0, 3, 1, 2), "conv1", stride=2, padding=3), "norm1"))
    for layer, stride in (("layer1", 1), ("layer2", 2), ("layer3", 2)):
        for i, st in ((0, stride), (1, 1)):
            pre = f"{layer}.{i}."
            y = F.relu(norm(cv(x, pre + "conv1", stride=st, padding=1), pre + "norm1"))
            y = F.relu(norm(cv(y, pre + "conv2", padding=1), pre + "norm2"))
            if st != 1:
                x = norm(cv(x, pre + "downsample.0", stride=st), pre + "norm3")
            x = F.relu(x + y)
    ref = cv(x, "conv2").permute(0, 2, 3, 1)
    enc = raft._Encoder(p, "group", backend)
    out = torch.empty(2, hw[0] // 8, hw[1] // 8, 256, device=backend)
    enc(frames.to(backend), out, split_tanh_relu=False)
    assert (out.double().cpu() - ref).abs().max() <= 2e-3 * ref.abs().max()
    with pytest.raises(ValueError, match="norm"):
        raft._Encoder(p, "layer", backend)


# --------------------------------------------------------------------------------------------
# streams, graphs, sizes (MI355X)
# --------------------------------------------------------------------------------------------
def _calls(dev, seed):
    """One call of each operator on inputs of its own -> (function, its outputs)."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, 24, 20, 320, generator=g).to(F16).to(dev)
    y = torch.empty_like(x)
    q, k, v = (torch.randn(90, n, 64, generator=g).to(BF16).to(dev) for n in (8, 2, 2))
    out, cu = torch.empty_like(q), _cu([50, 0, 40], dev)
    pq, ko, vo = torch.randn(3, 1, 8, 64, generator=g).to(BF16).to(dev), *(torch.randn(3, 70, 2, 64, generator=g).to(BF16).to(dev) for _ in range(2))
    po, n = torch.empty_like(pq), torch.tensor([70, 1, 33], dtype=torch.int32, device=dev)

    def run():
        ops.groupnorm(x, y, 32, act="silu")
        ops.prompt_attention(q, k, v, out, cu)
        ops.prefix_attention(pq, k, v, ko, vo, n, po)

    return run, (x, q, pq, ko), (y, out, po)


@gpu_only
def test_captured_and_replayed(hip_lib):
    """Two graphs of the same operators, replayed in turn on changing inputs with eager calls between: every replay equals the eager result
    bit for bit (no atomics, scratch of their own)."""
    dev = torch.device("cuda:0")
    both = [_calls(dev, s) for s in (31, 32)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for run, _, _ in both:
            run()
    side.synchronize()
    graphs = []
    for run, _, _ in both:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        graphs.append(graph)
    for rep in range(4):
        for (run, ins, outs), graph in zip(both, graphs):
            for t in ins:
                t.mul_(0.9)
            run()
            want = [t.clone() for t in outs]
            for t in outs:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(want, outs):
                assert torch.equal(a, b), rep


@gpu_only
def test_two_streams_at_once(hip_lib):
    dev = torch.device("cuda:0")
    calls = [_calls(dev, s) for s in (41, 42)]
    for run, _, _ in calls:
        run()
    torch.cuda.synchronize()
    want = [[t.clone() for t in outs] for _, _, outs in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(10):
        for st, (run, _, _) in zip(streams, calls):
            with torch.cuda.stream(st):
                run()
    torch.cuda.synchronize()
    for w, (_, _, outs) in zip(want, calls):
        for a, b in zip(w, outs):
            assert torch.equal(a, b)


@gpu_only
def test_long_and_wide(hip_lib):
    """Key offsets past 2^32 elements, a long prompt, a long prefix: against f32 products of torch on a few rows."""
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(51)
    kh, d, t = 2, 128, 700
    big_k, big_v = (torch.empty(t, 1 << 23, dtype=F16, device=dev) for _ in range(2))      # 11.7 GB each: row 512 starts past 2^32
    k, v = big_k[:, :kh * d].unflatten(1, (kh, d)), big_v[:, :kh * d].unflatten(1, (kh, d))
    k.copy_(torch.randn(t, kh, d, device=dev, generator=g))
    v.copy_(torch.randn(t, kh, d, device=dev, generator=g))
    q = torch.randn(t, 8, d, device=dev, generator=g).to(F16)
    out, same = torch.empty_like(q), torch.empty_like(q)
    cu = _cu([t], dev)
    ops.prompt_attention(q, k, v, out, cu)
    ops.prompt_attention(q, k.contiguous(), v.contiguous(), same, cu)
    assert torch.equal(out, same)
    own_k, own_v = k[None, :1].contiguous(), v[None, :1].contiguous()
    one = torch.empty(1, 8, d, dtype=F16, device=dev)
    ops.prefix_attention(q[-1:], k, v, own_k, own_v, torch.zeros(1, dtype=torch.int32, device=dev), one)
    tol = 4 * U[F16] * v.float().abs().max()
    assert (one[0] - out[-1]).abs().max() <= tol         # the last token of the prompt sees the same keys
    del big_k, big_v, k, v
    torch.cuda.empty_cache()
    n = 20000
    q, k, v = (torch.randn(n, h, 64, device=dev, generator=g).to(BF16) for h in (4, 1, 1))
    out = torch.empty_like(q)
    ops.prompt_attention(q, k, v, out, _cu([n], dev))
    for row in (0, 31, 32, 9999, n - 1):
        o, amp, _, smax = _attend_ref(q[row:row + 1].double().cpu(), k[:row + 1].double().cpu(), v[:row + 1].double().cpu(),
                                      torch.ones(1, row + 1, dtype=torch.bool), 64 ** -0.5)
        _within(out[row:row + 1], o, _attn_tol(BF16, o, amp, row + 1, 64, smax, v.float().abs().max().item()), row)


@gpu_only
@DT
@pytest.mark.parametrize("h,kh,d,lens,causal", [
    (8, 2, 64, [1000, 3, 517], True), (4, 4, 128, [300, 290], False), (6, 2, 96, [257, 128, 129], True), (2, 1, 256, [200, 310], True),
    (3, 1, 32, [700], True), (16, 1, 80, [100, 33], True)])
def test_prompt_attention_through_the_steady_state(hip_lib, dt, h, kh, d, lens, causal):
    """Sequences of many key blocks: the pipelined steps, both parities of their number, rising and falling maxima."""
    _check_prompt(torch.device("cuda:0"), dt, h, kh, d, lens, lens, causal)


@DT
@pytest.mark.parametrize("rising", [True, False])
def test_prompt_attention_with_moving_maxima(backend, dt, rising):
    """Scores that rise (or fall) by hundreds along the keys: the maximum has to move (or stay) in every block."""
    g = torch.Generator().manual_seed(61)
    n, d = 230, 32
    q = torch.randn(n, 1, d, generator=g) * 0.05 + 1
    k = torch.randn(n, 1, d, generator=g) * 0.05 + (torch.arange(n) if rising else torch.arange(n).flip(0))[:, None, None] * 0.1
    v = torch.randn(n, 1, d, generator=g)
    q, k, v = (t.to(dt).to(backend) for t in (q, k, v))
    for causal in (False, True):
        out = torch.empty_like(q)
        ops.prompt_attention(q, k, v, out, _cu([n], backend), causal=causal, scale=1.0)
        o, amp, _, smax = _attend_ref(q.double().cpu(), k.double().cpu(), v.double().cpu(), _seen(n, n, causal), 1.0)
        _within(out, o, _attn_tol(dt, o, amp, n, d, smax, v.float().abs().max().item()))
