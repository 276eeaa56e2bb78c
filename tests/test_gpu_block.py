"""Windowed attention and gated norms (block.py) against their definitions in 64 bits.

Tolerances are bounds, element by element, computed beside the reference.  With h = half a step of the type (bf16 2^-8, fp32 2^-24, relative):
  out:  h (sum p |v| [P rounded in front of its product] + |out| [rounded at the end]) + e32
  delta = dout . out uses the rounded out:  E_i = sum_d |dout| (out's bound)
  dv:   h (sum p |dout| + |dv|) + e32;   dq: scale sum_j (h |ds'_ij| + p_ij E_i) |k_j| + h |dq| + e32, ds' = p (dp - delta); dk likewise over i
e32: the same sums times the relative error of a probability computed in fp32, e_p = 2^-24 (2 dh S + 2 |s| + 8) with S = scale sum |q||k| (a dot product of n
terms is off by at most n 2^-24 of its absolute sum, exp2's argument is rounded, v_exp is good to 2^-23), plus 2^-24 times the number of terms that a sum adds."""
import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
dic = importlib.import_module("diffusion-image-captioning_amd")

BF16, F32 = torch.bfloat16, torch.float32
H = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
INF = math.inf


# ------------------------------------------------------------------------------------------------ attention: the definition
def visible(N, Tq, Tk, left, right, sinks, key_mask, kv_len, q_pos):
    i, j = torch.arange(Tq)[:, None], torch.arange(Tk)[None]
    see = torch.zeros(N, Tq, Tk, dtype=torch.bool)
    for n in range(N):
        t = i + (0 if q_pos is None else int(q_pos[n]))
        ok = torch.ones(Tq, Tk, dtype=torch.bool)
        if right is not None:
            ok &= j <= t + right
        if left is not None:
            ok &= (j >= t - left) | (j < sinks)
        if kv_len is not None:
            ok &= j < int(kv_len[n])
        if key_mask is not None:
            ok &= key_mask[n][None].cpu().bool()
        see[n] = ok
    return see.cuda()


def definition(q, k, v, see, scale, dout=None):
    """Values and bounds in 64 bits: {name: (value, bound)}; hidden rows of k and v count as zero."""
    h = H[q.dtype]
    G = q.shape[2] // k.shape[2]
    dead = ~see.any(1)                                                     # [N, Tk]
    k, v = (t.double().masked_fill(dead[:, :, None, None], 0.0) for t in (k, v))
    Q = q.double().transpose(1, 2)
    K, V = (t.transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
    at = lambda a, b: torch.matmul(a, b.transpose(2, 3).contiguous())      # noqa: E731
    vis = see[:, None]
    s = (at(Q, K) * scale).masked_fill(~vis, -INF)
    big = at(Q.abs(), K.abs()) * scale
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -INF, torch.zeros_like(m), m)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    p = torch.where(z > 0, e / torch.where(z > 0, z, torch.ones_like(z)), torch.zeros_like(e))
    lse = (m + z.log())[..., 0]
    s = s.masked_fill(~vis, 0.0)
    n = max(s.shape[-1], s.shape[-2] * G, 8)
    ep = 2.0 ** -24 * (2 * q.shape[3] * big.amax((-1, -2), keepdim=True) + 2 * s.abs().amax((-1, -2), keepdim=True) + 8 + n)
    o = torch.matmul(p, V)
    pv = torch.matmul(p, V.abs())
    bo = h * (pv + o.abs()) + 2 * ep * pv
    got = {"out": (o.transpose(1, 2), bo.transpose(1, 2)), "lse": (lse, (ep[..., 0] + 2.0 ** -22) * (1 + torch.nan_to_num(lse, neginf=0.0).abs()))}
    if dout is None:
        return got
    D = dout.double().transpose(1, 2)
    fold = lambda t: t.view(t.shape[0], t.shape[1] // G, G, *t.shape[2:]).sum(2).transpose(1, 2)   # noqa: E731
    tr = lambda t: t.transpose(2, 3).contiguous()                                                  # noqa: E731
    dv, adv = torch.matmul(tr(p), D), torch.matmul(tr(p), D.abs())
    dp, delta = at(D, V), (D * o).sum(-1, keepdim=True)
    big_dp = at(D.abs(), V.abs())
    E = (D.abs() * bo).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    b = h * ds.abs() + p * (E + 2.0 ** -24 * q.shape[3] * (big_dp + (D.abs() * o.abs()).sum(-1, keepdim=True))) + 2 * ep * p * (dp.abs() + delta.abs())
    dq, dk = torch.matmul(ds, K) * scale, torch.matmul(tr(ds), Q) * scale
    eb = 2.0 ** -24 * n * ds.abs()
    bq = torch.matmul(b + eb, K.abs()) * scale + h * dq.abs()
    bk, bv = torch.matmul(tr(b + eb), Q.abs()) * scale, (h + 2 * ep.transpose(2, 3)) * adv
    dk, dv = fold(dk), fold(dv)
    got["dq"] = (dq.transpose(1, 2), bq.transpose(1, 2))
    got["dk"] = (dk, fold(bk) + h * dk.abs())
    got["dv"] = (dv, fold(bv) + h * dv.abs())
    return got


def holds(name, got, want):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    x = got.double()
    same = (x == value) | (torch.isinf(value) & (x == value))
    off = (x - value).abs()
    bad = ~(same | (off <= bound + 1e-30))
    assert not bad.any(), (name, int(bad.sum()), float(off[bad].nan_to_num(INF).max()), [float(t) for t in (x[bad][0], value[bad][0], bound.expand_as(value)[bad][0])])
    fine = torch.isfinite(value)
    # Rounding errors of fp32 that are as good as independent stay far below the bound of the worst case.  (A row that sees one key has p = 1 and ds =
    # dp - delta = 0: where no row sees more, dq and dk are nothing but rounding, 64 bits included, and only the bound says something: values below 2^-40.)
    if got.dtype == F32 and name != "lse" and fine.any() and float(value[fine].abs().max()) > 2.0 ** -40:
        assert float((x - value)[fine].norm() / value[fine].norm()) < 2e-5, name


CASES = {
    # name: N, Tq, Tk, H, Hkv, dh, left, right, sinks
    "one key": (2, 1, 1, 3, 3, 64, None, None, 0),
    "one query": (3, 1, 77, 4, 2, 64, None, 0, 0),
    "31": (1, 31, 31, 2, 2, 64, 5, 5, 1),
    "32": (2, 32, 32, 2, 1, 128, 5, 0, 2),
    "33": (1, 33, 33, 2, 2, 64, None, 0, 0),
    "64": (1, 64, 64, 1, 1, 64, 16, None, 3),
    "65": (2, 65, 65, 4, 4, 64, 20, 20, 2),
    "127": (1, 127, 127, 2, 2, 128, 30, 7, 0),
    "129": (1, 129, 129, 3, 1, 64, 63, 0, 4),
    "only itself": (1, 100, 100, 2, 2, 64, 0, 0, 0),
    "itself and sinks": (1, 300, 300, 2, 2, 64, 0, 0, 5),
    "sinks over a tile": (1, 300, 300, 2, 1, 128, 10, 0, 70),
    "more sinks than keys": (1, 40, 40, 2, 2, 64, 3, 0, 1000),
    "no window": (2, 200, 200, 2, 2, 64, None, None, 0),
    "long, causal": (1, 700, 700, 8, 2, 128, 200, 0, 4),
    "long, both sides": (2, 530, 530, 3, 3, 64, 100, 60, 2),
    "many keys, few queries": (2, 5, 1000, 8, 1, 128, None, 0, 0),
    "few keys, many queries": (2, 400, 20, 2, 2, 64, 50, None, 2),
    "group of 8": (1, 150, 150, 16, 2, 64, 40, 0, 1),
    "every query sees far keys": (1, 1500, 1500, 2, 1, 64, 10, 0, 3),
    "many far keys, wide rows": (2, 1100, 1100, 4, 2, 128, 20, 5, 70),
    "one query, keys for several workgroups": (1, 1, 3000, 2, 2, 64, None, 0, 0),
    "32 rows, keys for several workgroups": (1, 8, 2000, 8, 2, 128, 1500, 0, 40),
    "256 rows and keys": (2, 256, 256, 2, 2, 64, 100, 100, 2),
    "257 rows and keys": (1, 257, 257, 2, 2, 64, 100, 100, 2),
    "many short sequences": (300, 40, 40, 2, 1, 64, 12, 12, 1),
    "many sequences, wide rows": (140, 130, 130, 2, 2, 128, 50, 0, 2),
    "heads of one workgroup": (130, 100, 70, 2, 2, 64, 20, 30, 1),
    "heads of one workgroup, 128 rows": (128, 128, 128, 2, 2, 64, None, None, 0),
    "heads of one workgroup, wide rows": (86, 200, 224, 3, 3, 128, 60, 0, 2),
    "heads of one workgroup, few queries": (256, 3, 120, 1, 1, 128, None, 100, 0),
    "wide rows, many keys": (1, 70, 2100, 2, 1, 128, None, None, 0),
    "many workgroups": (20, 290, 290, 8, 4, 64, 60, 0, 2),
    "many workgroups, wide rows": (16, 300, 300, 8, 2, 128, 100, 20, 1),
    "many workgroups, many keys": (5, 140, 2100, 26, 13, 128, None, None, 0),
    "wide rows, windows over 2000 keys": (1, 2300, 2300, 1, 1, 128, 2060, 0, 3),
}


def run_both(dtype, shape, *, key_mask=None, kv_len=None, q_pos=None, scale=None, seed=0, spoil=False, views=False):
    N, Tq, Tk, Hq, Hkv, dh, left, right, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)   # noqa: E731
    if views:                                                                # rows of one packed tensor, longer than what is read
        packed = new(N, max(Tq, Tk) + 3, Hq + 2 * Hkv, dh)
        q, k, v = packed[:, :Tq, :Hq], packed[:, 1:Tk + 1, Hq:Hq + Hkv], packed[:, 2:Tk + 2, Hq + Hkv:]
        dout = new(N, Hq, Tq, dh).transpose(1, 2)
    else:
        q, k, v, dout = new(N, Tq, Hq, dh), new(N, Tk, Hkv, dh), new(N, Tk, Hkv, dh), new(N, Tq, Hq, dh)
    see = visible(N, Tq, Tk, left, right, sinks, key_mask, kv_len, q_pos)
    want = definition(q, k, v, see, scale or dh ** -0.5, dout)
    if spoil:                                                                # what nobody may see holds anything
        dead = torch.zeros(N, Tk, dtype=torch.bool, device="cuda")
        if kv_len is not None:
            dead |= torch.arange(Tk, device="cuda")[None] >= kv_len[:, None]
        if key_mask is not None:
            dead |= ~key_mask.bool()
        k[dead], v[dead] = math.nan, INF
    how = dict(left=left, right=right, sinks=sinks, key_mask=key_mask, kv_len=kv_len, q_pos=q_pos, scale=scale)
    out, lse = dic.window_attention(q, k, v, **how)
    holds("out", out, want["out"])
    holds("lse", lse, want["lse"])
    for name, t in zip(("dq", "dk", "dv"), dic.window_attention_grad(dout, q, k, v, out, lse, **how)):
        holds(name, t, want[name])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", CASES)
def test_window_attention(case, dtype):
    run_both(dtype, CASES[case], seed=len(case))


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("dh", [64, 128])
def test_window_attention_reads_views_of_packed_tensors(dtype, dh):
    run_both(dtype, (2, 90, 75, 4, 2, dh, 30, 10, 3), views=True, scale=0.3)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Tq", [1, 3, 140])
def test_keys_that_nobody_may_see_are_not_read_into_results(dtype, Tq):
    N, Tk = 5, 140
    lens = torch.tensor([Tk, 0, 1, 77, 400], dtype=torch.int32, device="cuda")         # (longer than the cache: all of it)
    mask = torch.rand(N, Tk, generator=torch.Generator().manual_seed(3)).cuda() < 0.6
    mask[3] = False
    for key_mask, kv_len in ((mask, None), (None, lens), (mask.to(torch.uint8), lens)):
        for left, right in ((None, None), (20, 0), (9, 30)):
            run_both(dtype, (N, Tq, Tk, 4, 2, 64, left, right, 2), key_mask=key_mask, kv_len=kv_len, spoil=True)


WIDE = {
    # N, Tq, Tk, H, Hkv, dh, left, right, sinks: spans of more than 2000 keys, in many workgroups (of 128 wide rows: tiles of 32 keys) and in few
    "many workgroups, window": (5, 140, 2600, 26, 13, 128, 2100, 30, 5), "many workgroups, causal": (5, 140, 2600, 26, 2, 128, None, 0, 0),
    "many workgroups, sinks over a tile": (5, 129, 2500, 26, 26, 128, 2060, 0, 70), "many workgroups, 64 wide": (5, 140, 2600, 26, 13, 64, 2100, 30, 5),
    "few workgroups": (5, 140, 2600, 2, 1, 128, 2100, 30, 5), "few rows": (5, 4, 2600, 8, 1, 128, 2100, 30, 5), "whole text": (1, 2300, 2300, 2, 1, 128, 2060, 0, 3),
}


@pytest.mark.parametrize("hidden", ["nothing", "a mask", "lengths and positions", "all of them"])
@pytest.mark.parametrize("case", WIDE)
def test_wide_windows_in_bf16(case, hidden):
    """Besides the bounds, which are wide here, the norms: P or ds, the result, and with dq and dk `out` behind delta are rounded, each by at most h = 2^-8 and, evenly
    spread, h / sqrt 3 in the mean square: h together.  A key too many or too few at the edge of n changes a row by about 1 / sqrt n of its norm, 0.02 here
    (0.003 of the whole text, whose first rows carry most of its norm)."""
    N, Tq, Tk, Hq, Hkv, dh, left, right, sinks = WIDE[case]
    g = torch.Generator(device="cuda").manual_seed(Tq + dh)
    q, k, v, dout = (torch.randn(N, t, n, dh, generator=g, device="cuda").to(BF16) for t, n in ((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq)))
    mask = torch.rand(N, Tk, generator=g, device="cuda") < 0.9 if hidden in ("a mask", "all of them") else None
    lens, pos = None, torch.full((N,), Tk - Tq, dtype=torch.int32, device="cuda")
    if hidden in ("lengths and positions", "all of them"):
        lens = torch.tensor([Tk, Tk - 1, Tk - 33, Tk - 64, Tk // 2][:N], dtype=torch.int32, device="cuda")
        pos = torch.tensor([Tk - Tq, Tk - Tq - 1, Tk - Tq - 40, 0, Tk // 2 - Tq][:N], dtype=torch.int32, device="cuda")
    how = dict(left=left, right=right, sinks=sinks, key_mask=mask, kv_len=lens, q_pos=pos)
    want = definition(q, k, v, visible(N, Tq, Tk, left, right, sinks, mask, lens, pos), dh ** -0.5, dout)
    out, lse = dic.window_attention(q, k, v, **how)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *dic.window_attention_grad(dout, q, k, v, out, lse, **how))):
        holds(name, t, want[name])
        if name != "lse":
            value = want[name][0]
            assert float((t.double() - value).norm() / value.norm()) < 2.0 ** -8, name


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("N,H,dh", [(24, 8, 64), (24, 6, 128), (3, 2, 64), (3, 2, 128)])
def test_many_and_few_workgroups_with_masks_lengths_and_positions(dtype, N, H, dh):
    """Odd numbers of key tiles, for workgroups that share them between their waves and for those that do not."""
    T = 310
    g = torch.Generator().manual_seed(N + dh)
    lens = torch.randint(0, T + 1, (N,), generator=g, dtype=torch.int32).cuda()
    mask = (torch.rand(N, T, generator=g) < 0.7).cuda()
    mask[1] = False
    pos = torch.randint(-100, 100, (N,), generator=g, dtype=torch.int32).cuda()
    run_both(dtype, (N, T, T, H, 2, dh, 70, 30, 5), key_mask=mask, kv_len=lens, q_pos=pos, spoil=True)
    run_both(dtype, (N, T, T, H, 2, dh, None, 0, 0), key_mask=mask, spoil=True)
    run_both(dtype, (N, T, 300, H, 2, dh, None, None, 0), kv_len=lens, spoil=True)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Tq,H,Hkv", [(1, 4, 2), (5, 2, 2), (40, 2, 2), (40, 4, 2), (150, 2, 1)])
def test_keys_outside_of_every_window_are_not_read_into_results(dtype, Tq, H, Hkv):
    """Rows of a cache in front of its newest token, and between the first keys and the oldest window, hold anything."""
    N, Tk = 4, 333
    pos = torch.tensor([0, 40, 170, Tk - Tq], dtype=torch.int32, device="cuda")
    for left, right, sinks in ((None, 0, 0), (20, 0, 3), (70, 7, 40), (9, None, 2), (0, 0, 0)):
        g = torch.Generator(device="cuda").manual_seed(Tq)
        q, k, v, dout = (torch.randn(N, t, h, 64, generator=g, device="cuda").to(dtype) for t, h in ((Tq, H), (Tk, Hkv), (Tk, Hkv), (Tq, H)))
        see = visible(N, Tq, Tk, left, right, sinks, None, None, pos.long())
        want = definition(q, k, v, see, 0.125, dout)
        dead = ~see.any(1)
        k[dead], v[dead] = math.nan, INF
        how = dict(left=left, right=right, sinks=sinks, q_pos=pos)
        out, lse = dic.window_attention(q, k, v, **how)
        for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *dic.window_attention_grad(dout, q, k, v, out, lse, **how))):
            holds(name, t, want[name])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Tq,Tk,dh", [(1, 40, 64), (60, 128, 64), (100, 33, 128), (128, 96, 128)])
def test_heads_of_one_workgroup_with_masks_lengths_and_positions(dtype, Tq, Tk, dh):
    """As many heads as let a workgroup take one whole in the backward pass, views of packed tensors, keys hidden in every way."""
    N = 132
    g = torch.Generator().manual_seed(Tq)
    lens = torch.randint(0, Tk + 40, (N,), generator=g, dtype=torch.int32).cuda()
    mask = (torch.rand(N, Tk, generator=g) < 0.7).cuda()
    mask[5] = False
    pos = torch.randint(-60, 60, (N,), generator=g, dtype=torch.int32).cuda()
    run_both(dtype, (N, Tq, Tk, 2, 2, dh, 20, 10, 3), key_mask=mask, kv_len=lens, q_pos=pos, views=True, spoil=True)
    run_both(dtype, (N, Tq, Tk, 2, 2, dh, None, None, 0), key_mask=mask, views=True, spoil=True)
    run_both(dtype, (N, Tq, Tk, 2, 2, dh, 30, None, 50), kv_len=lens, q_pos=pos, spoil=True)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_query_positions(dtype):
    """Rows far before, inside and far behind the keys; rows that see nothing."""
    pos = torch.tensor([-500, -40, 0, 100, 250, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    clamped = pos.clamp(-2 ** 29, 2 ** 29)
    for left, right, sinks in ((30, 0, 0), (30, 5, 2), (None, 0, 0), (30, None, 1)):
        N, Tq, Tk = len(pos), 50, 260
        g = torch.Generator(device="cuda").manual_seed(7)
        q, k, v, dout = (torch.randn(N, t, 2, 64, generator=g, device="cuda").to(dtype) for t in (Tq, Tk, Tk, Tq))
        how = dict(left=left, right=right, sinks=sinks, q_pos=pos)
        want = definition(q, k, v, visible(N, Tq, Tk, left, right, sinks, None, None, clamped.long()), 0.125, dout)
        out, lse = dic.window_attention(q, k, v, **how)
        for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *dic.window_attention_grad(dout, q, k, v, out, lse, **how))):
            holds(name, t, want[name])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Tq,Hq,Hkv", [(2, 4, 2), (50, 4, 2), (50, 2, 2)])
def test_bounds_as_far_as_the_farthest_positions(dtype, Tq, Hq, Hkv):
    """Finite bounds beside positions of +-2^29: they cut where they say, and larger ones nowhere."""
    pos = torch.tensor([2 ** 29, 2 ** 29 - 7, 2 ** 31 - 1, 0, -2 ** 29, 7 - 2 ** 29, -2 ** 31], dtype=torch.int32, device="cuda")
    clamped = pos.clamp(-2 ** 29, 2 ** 29)
    N, Tk = len(pos), 260
    g = torch.Generator(device="cuda").manual_seed(7)
    q, k, v, dout = (torch.randn(N, t, n, 64, generator=g, device="cuda").to(dtype) for t, n in ((Tq, Hq), (Tk, Hkv), (Tk, Hkv), (Tq, Hq)))
    for left, right in ((2 ** 31 - 1, None), (None, 2 ** 31 - 1), (2 ** 30, 2 ** 30), (2 ** 31 - 1, 0), (2 ** 29, None), (2 ** 29 - 100, 2 ** 29 + 90), (None, 2 ** 29 + 3)):
        how = dict(left=left, right=right, sinks=2, q_pos=pos)
        want = definition(q, k, v, visible(N, Tq, Tk, left, right, 2, None, None, clamped.long()), 0.125, dout)
        out, lse = dic.window_attention(q, k, v, **how)
        for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *dic.window_attention_grad(dout, q, k, v, out, lse, **how))):
            holds(name, t, want[name])


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("Tq", [2, 60])
def test_masks_of_more_tiles_than_are_read_at_once(dtype, Tq):
    """A mask over 35000 keys (547 tiles of 64, 1094 of 32), most of them hidden; the queries stand at the end."""
    Tk = 35000
    mask = torch.rand(1, Tk, generator=torch.Generator().manual_seed(9)).cuda() < 0.3
    pos = torch.tensor([Tk - Tq], dtype=torch.int32, device="cuda")
    run_both(dtype, (1, Tq, Tk, 1, 1, 64, None, 0, 0), key_mask=mask, q_pos=pos, spoil=True)
    run_both(dtype, (1, Tq, Tk, 1, 1, 64, 30000, 0, 5), key_mask=mask, q_pos=pos, spoil=True)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
def test_far_keys_with_masks_lengths_and_positions(dtype):
    """Keys that all queries see beside windows of 25, where some of them are hidden, or behind a sequence's end, or the queries start elsewhere."""
    N, T = 3, 900
    mask = torch.ones(N, T, dtype=torch.bool, device="cuda")
    mask[1, 3:20] = False
    lens = torch.tensor([T, 700, 9], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 40, -30], dtype=torch.int32, device="cuda")
    run_both(dtype, (N, T, T, 2, 1, 64, 20, 4, 40), key_mask=mask, kv_len=lens, q_pos=pos, spoil=True)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T", [50, 400])
def test_large_logits(dtype, T):
    """Logits in the hundreds: the maximum moves far from tile to tile, most probabilities vanish."""
    g = torch.Generator(device="cuda").manual_seed(T)
    q, k, v, dout = (torch.randn(1, T, 2, 64, generator=g, device="cuda").to(dtype) for _ in range(4))
    ramp = torch.linspace(-1, 1, T, device="cuda").view(1, T, 1, 1)
    k = (k * 4 + 20 * ramp * torch.sign(q.mean(1, keepdim=True))).to(dtype)
    want = definition(q, k, v, visible(1, T, T, None, 0, 0, None, None, None), 1.0, dout)
    out, lse = dic.window_attention(q, k, v, right=0, scale=1.0)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *dic.window_attention_grad(dout, q, k, v, out, lse, right=0, scale=1.0))):
        value, bound = want[name]
        off = (t.double() - value).abs()
        assert (off <= bound + 1e-30).all(), (name, float((off - bound).max()))


@pytest.mark.parametrize("shape", [(64, 100, 100, 2, 2, 64, 2, 0, 0), (2, 900, 900, 4, 2, 64, 2, 0, 0), (2, 900, 900, 4, 2, 128, 3, 0, 1), (128, 17, 17, 4, 4, 64, None, None, 0),
                                   (130, 17, 17, 2, 2, 128, None, None, 0), (30, 17, 17, 4, 2, 64, None, None, 0)])
def test_few_keys_share_a_row_and_its_gradients_are_as_good_as_two_roundings(shape):
    """bf16 gradients of narrow windows: ds is rounded and so is the result, each by at most h = 2^-8 of a value and, evenly spread, h / sqrt 3 in the mean square.
    The rounding of `out` must not add to that through dout . out (it did: 0.0037 of the norm, where h sqrt(2 / 3) = 0.0032)."""
    N, Tq, Tk, Hq, Hkv, dh, left, right, sinks = shape
    g = torch.Generator(device="cuda").manual_seed(Tq)
    q, k, v, dout = (torch.randn(N, Tq, h, dh, generator=g, device="cuda").to(BF16) for h in (Hq, Hkv, Hkv, Hq))
    want = definition(q, k, v, visible(N, Tq, Tk, left, right, sinks, None, None, None), dh ** -0.5, dout)
    how = dict(left=left, right=right, sinks=sinks)
    out, lse = dic.window_attention(q, k, v, **how)
    for name, t in zip(("dq", "dk", "dv"), dic.window_attention_grad(dout, q, k, v, out, lse, **how)):
        value = want[name][0]
        assert float((t.double() - value).norm() / value.norm()) < 2.0 ** -8 * math.sqrt(2 / 3), name


def gradients_of_peaked_rows(left, sinks, mask, scale):
    """bf16 dq, dk, dv and their exact values for 2 x 900 rows, 4 query and 2 key heads, causal: logits spread widely enough that a few keys hold a row's weight."""
    N, T, Hq, Hkv, dh = 2, 900, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(T)
    q, k, v, dout = (torch.randn(N, T, h, dh, generator=g, device="cuda").to(BF16) for h in (Hq, Hkv, Hkv, Hq))
    how = dict(left=left, right=0, sinks=sinks, key_mask=mask, scale=scale)
    want = definition(q, k, v, visible(N, T, T, left, 0, sinks, mask, None, None), scale, dout)
    out, lse = dic.window_attention(q, k, v, **how)
    return dict(zip(("dq", "dk", "dv"), dic.window_attention_grad(dout, q, k, v, out, lse, **how))), {k: want[k][0] for k in ("dq", "dk", "dv")}


def test_sinks_inside_the_window_count_once_where_few_keys_share_a_row():
    """Rows 128 to 255 of a causal text see at most 256 keys, all inside the window, the sinks among them: as good as two roundings (above)."""
    got, want = gradients_of_peaked_rows(500, 400, None, 0.6)
    part = slice(128, 256)
    assert float((got["dq"].double() - want["dq"])[:, part].norm() / want["dq"][:, part].norm()) < 2.0 ** -8 * math.sqrt(2 / 3)


@pytest.mark.parametrize("left,sinks,every", [(None, 0, 4), (600, 0, 200), (600, 5, 200), (300, 600, 4), (400, 40, 9)])
def test_few_keys_that_a_mask_leaves_share_a_row(left, sinks, every):
    """Long spans of which key_mask leaves at most 256 keys: as good as two roundings, as if there were no others."""
    mask = torch.zeros(2, 900, dtype=torch.bool, device="cuda")
    mask[:, ::every] = True
    got, want = gradients_of_peaked_rows(left, sinks, mask, 0.6)
    for name in got:
        assert float((got[name].double() - want[name]).norm() / want[name].norm()) < 2.0 ** -8 * math.sqrt(2 / 3), name


@pytest.mark.parametrize("Tq,Tk", [(0, 5), (5, 0), (0, 0)])
def test_window_attention_of_nothing(Tq, Tk):
    q, k = torch.randn(2, Tq, 4, 64, device="cuda"), torch.randn(2, Tk, 2, 64, device="cuda")
    out, lse = dic.window_attention(q, k, k, left=3, right=3, sinks=1)
    dq, dk, dv = dic.window_attention_grad(torch.ones_like(q), q, k, k, out, lse, left=3, right=3, sinks=1)
    assert out.shape == q.shape and not out.any() and (lse == -INF).all()
    assert not dq.any() and not dk.any() and not dv.any() and dk.shape == dv.shape == k.shape
    none = dic.window_attention(q[:0], k[:0], k[:0])[0]
    assert none.shape == (0, Tq, 4, 64)


def test_window_attention_gradients_are_differences_of_the_output():
    """Along random directions: (f(t + e) - f(t - e)) / 2 e of f = sum(out * dout), in 64 bits on the definition's side, against the fp32 kernels' gradients."""
    N, T, Hq, Hkv, dh = 1, 45, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(5)
    q, k, v, dout = (torch.randn(N, T, n, dh, generator=g, device="cuda") for n in (Hq, Hkv, Hkv, Hq))
    how = dict(left=7, right=2, sinks=3)
    see = visible(N, T, T, 7, 2, 3, None, None, None)
    out, lse = dic.window_attention(q, k, v, **how)
    grads = dic.window_attention_grad(dout, q, k, v, out, lse, **how)
    for which in range(3):
        args = [q.double(), k.double(), v.double()]
        u = torch.randn(args[which].shape, generator=g, device="cuda", dtype=torch.float64)
        f = []
        for e in (1e-4, -1e-4):
            moved = list(args)
            moved[which] = args[which] + e * u
            s = torch.matmul(moved[0].transpose(1, 2), moved[1].transpose(1, 2).repeat_interleave(2, 1).transpose(2, 3).contiguous()) * dh ** -0.5
            o = torch.matmul(torch.softmax(s.masked_fill(~see[:, None], -INF), -1), moved[2].transpose(1, 2).repeat_interleave(2, 1))
            f.append(float((o.transpose(1, 2) * dout.double()).sum()))
        slope = (f[0] - f[1]) / 2e-4
        assert abs(slope - float((grads[which].double() * u).sum())) < 1e-4 * (1 + abs(slope))      # 2e-5 of the norm, and e^2 of the differences


@pytest.mark.parametrize("Tq,Tk,Hq", [(1, 300, 4), (200, 300, 2), (100, 230, 1), (290, 300, 1)])
def test_rows_of_a_cache_far_apart(Tq, Tk, Hq):
    """Tokens 16 MiB apart, so that offsets pass 2^32 bytes: the results of the same rows side by side, bit for bit."""
    step = 1 << 23                                                           # bf16 elements
    g = torch.Generator(device="cuda").manual_seed(Tk)
    q, dout = (torch.randn(1, Tq, Hq, 64, generator=g, device="cuda").to(BF16) for _ in range(2))
    k, v = (torch.randn(1, Tk, 1, 64, generator=g, device="cuda").to(BF16) for _ in range(2))
    room = torch.empty(step * (Tk - 1) + 256, dtype=BF16, device="cuda")
    far = [room.as_strided((1, Tk, 1, 64), (0, step, 0, 1), 64 * i) for i in range(4)]
    far[0].copy_(k)
    far[1].copy_(v)
    for how in (dict(left=120, right=0, sinks=3, q_pos=torch.tensor([Tk - Tq], dtype=torch.int32, device="cuda")), dict()):
        out, lse = dic.window_attention(q, k, v, **how)
        dq, dk, dv = dic.window_attention_grad(dout, q, k, v, out, lse, **how)
        o2, l2 = dic.window_attention(q, *far[:2], **how)
        d2 = torch.empty_like(q)
        dic.window_attention_grad(dout, q, *far[:2], o2, l2, grads=(d2, far[2], far[3]), **how)
        for name, x, y in (("out", out, o2), ("lse", lse, l2), ("dq", dq, d2), ("dk", dk, far[2]), ("dv", dv, far[3])):
            assert torch.equal(x, y), name


def test_outputs_can_be_views_and_nothing_else_is_written():
    N, T, Hq, Hkv, dh = 2, 70, 4, 2, 64
    qkv = torch.randn(N, T, Hq + 2 * Hkv, dh, device="cuda").to(BF16)
    q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    room = torch.full((N, T + 2, Hq, dh + 8), 7.0, device="cuda", dtype=BF16)
    out, lse = dic.window_attention(q, k, v, left=9, right=9, out=room[:, 1:-1, :, :dh])
    plain, _ = dic.window_attention(q, k, v, left=9, right=9)
    assert torch.equal(out, plain) and (room[:, 0] == 7).all() and (room[:, -1] == 7).all() and (room[..., dh:] == 7).all()
    dout = torch.randn_like(plain)
    dqkv = torch.full((N, T, Hq + 2 * Hkv + 1, dh), 7.0, device="cuda", dtype=BF16)
    parts = dqkv[:, :, :Hq], dqkv[:, :, Hq:Hq + Hkv], dqkv[:, :, Hq + Hkv:-1]
    dic.window_attention_grad(dout, q, k, v, out, lse, left=9, right=9, grads=parts)
    for a, b in zip(parts, dic.window_attention_grad(dout, q, k, v, plain, lse, left=9, right=9)):
        assert torch.equal(a, b)
    assert (dqkv[:, :, -1] == 7).all()


# ------------------------------------------------------------------------------------------------ norms
def norm_definition(v, kind, w, b, eps):
    """(normed, mean, rstd) of rows in 64 bits."""
    zero = torch.zeros(v.shape[0], 1, dtype=torch.float64, device=v.device)
    if kind == "none":
        return v, zero, zero
    mean = v.mean(1, keepdim=True) if kind == "layer" else zero
    rstd = ((v - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    u = (v - mean) * rstd
    u = u * w.double() if w is not None else u
    return (u + b.double() if b is not None else u), mean, rstd


def close32(name, got, want, scale, terms):
    """fp32 arithmetic over `terms` additions of numbers whose absolute sum is `scale`: off by at most (terms + 16) 2^-24 of it."""
    off = (got.double() - want).abs()
    bound = (terms + 16) * 2.0 ** -24 * scale + 1e-30
    assert (off <= bound).all(), (name, float((off / bound).max()))


NORMS = [
    # sequences, rows each, D, gate, post, pre, bias
    (1, 1, 1, "shared", "rms", "rms", True), (2, 3, 5, "sequence", "layer", "rms", True), (1, 4, 63, None, "layer", "layer", False), (3, 7, 64, "sequence", "rms", "layer", True),
    (5, 1, 65, "sequence", "layer", "none", True), (2, 9, 127, "shared", "none", "layer", True), (40, 2, 128, "sequence", "layer", "layer", True), (2, 33, 255, "sequence", "layer", "layer", True),
    (1, 5, 256, None, "none", "rms", False), (7, 3, 511, "shared", "layer", "layer", True), (2, 8, 512, "sequence", "rms", "rms", False),
    (64, 17, 768, "sequence", "layer", "layer", True), (1, 2500, 768, "shared", "layer", "layer", True), (3, 1100, 767, "sequence", "layer", "rms", True),
    (2, 65, 1003, "sequence", "layer", "layer", True), (2, 6, 1024, "shared", "rms", "layer", True), (3, 50, 1500, "sequence", "layer", "layer", True), (1, 3, 2048, "shared", "layer", "layer", True),
    (2, 40, 4095, "sequence", "rms", "layer", True), (2, 3, 4096, None, "layer", "layer", True), (2, 30, 8191, "sequence", "layer", "rms", True), (1, 1300, 8192, "shared", "layer", "layer", False),
    (3000, 1, 96, "sequence", "layer", "layer", True), (1, 20000, 40, "shared", "layer", "rms", True), (9, 1111, 120, "sequence", "rms", "layer", True),
    (1100, 3, 200, "sequence", "layer", "layer", True), (700, 2, 770, "sequence", "layer", "rms", True), (520, 3, 1500, "sequence", "rms", "layer", True), (300, 2, 2500, "sequence", "layer", "layer", True),
    (260, 1, 5000, "sequence", "rms", "rms", True),
]
TYPES = [(F32, F32), (BF16, BF16), (F32, BF16)]


def norm_inputs(case, stream, inner, seed=0):
    N, T, D, gate, post, pre, bias = case
    g = torch.Generator(device="cuda").manual_seed(seed + D)
    new = lambda *s: torch.randn(*s, generator=g, device="cuda")             # noqa: E731
    x, y = (new(N, T, D) * 1.5 + 0.3).to(stream), (new(N, T, D) * 0.7 - 0.2).to(inner)
    norms = {side: dic.NormParams(kind, 1 + 0.1 * new(D), 0.1 * new(D) if bias else None, 1e-5) if kind != "none" else None for side, kind in (("post", post), ("pre", pre))}
    gt = {"sequence": lambda: new(N, D), "shared": lambda: new(D), None: lambda: None}[gate]()
    return x, y, norms, gt, new


@pytest.mark.parametrize("stream,inner", TYPES, ids=["fp32", "bf16", "fp32 stream"])
@pytest.mark.parametrize("case", NORMS, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}-{c[3]}-{c[4]}-{c[5]}")
def test_gated_norm(case, stream, inner):
    N, T, D, gate, post, pre, bias = case
    x, y, norms, g, new = norm_inputs(case, stream, inner)
    r = 0.75
    rows = lambda t: t.double().view(N * T, D)                               # noqa: E731
    get = lambda side, k: getattr(norms[side], k) if norms[side] is not None else None      # noqa: E731
    wide = torch.ones(N * T, D, dtype=torch.float64, device="cuda") if g is None else g.double().expand(N * T, D) if g.dim() == 1 else g.double().repeat_interleave(T, 0)
    n, m2, r2 = norm_definition(rows(y), post, get("post", "weight"), get("post", "bias"), 1e-5)
    v = r * rows(x) + wide * n
    a, m1, r1 = norm_definition(v, pre, get("pre", "weight"), get("pre", "bias"), 1e-5)
    x_new, got, saved = dic.gated_norm(x, y, gate=g, residual_scale=r, **norms)
    # a normed element: off by (D + 16) 2^-24 of |v| + |mean| + rms times rstd |w|, at most; deviations are >= 0.5 here except where D is small
    def spread(t, m, rs, w):
        return (t.abs() + m.abs() + t.square().mean(1, keepdim=True).sqrt()) * rs * (w.double().abs() if w is not None else 1.0) * (1 + (t - m).abs() * rs)
    en = rows(y).abs() if post == "none" else spread(rows(y), m2, r2, get("post", "weight")) + 1
    ev = (D + 16) * 2.0 ** -24 * (rows(x).abs() + wide.abs() * en)
    hx, hy = (0 if stream == F32 else 2.0 ** -8), (0 if inner == F32 else 2.0 ** -8)
    off = (rows(x_new) - v).abs()
    assert (off <= ev + hx * v.abs()).all(), float((off - ev - hx * v.abs()).max())
    if pre != "none":
        ea = ((D + 16) * 2.0 ** -24 * (spread(v, m1, r1, get("pre", "weight")) + 1)
              + 3 * ev.amax(1, keepdim=True) * r1 * (get("pre", "weight").double().abs() if get("pre", "weight") is not None else 1.0) * (1 + (v - m1).abs() * r1))
        off = (rows(got) - a).abs()
        assert (off <= ea + hy * a.abs()).all(), float((off - ea - hy * a.abs()).max())
        assert float((rows(got) - a).norm() / a.norm().clamp_min(1e-30)) < (2e-5 if inner == F32 and D > 1 else 2.0 ** -8 if D > 1 else INF)
    else:
        assert got is None
    for k, want in enumerate((m2, r2, m1, r1)):
        if D > 8:
            assert torch.allclose(saved[k].double(), want[:, 0], rtol=2e-5, atol=2e-6), k

    # gradients, from what the forward call left (its statistics are inputs here)
    dx_new, da = new(N, T, D).to(stream), new(N, T, D).to(inner) if pre != "none" else None
    back = dic.gated_norm_grad(dx_new, da, x_new, y, saved, gate=g, residual_scale=r, **norms)
    st = saved.double()[..., None]

    def norm_back(d, t, m, rs, w, kind):
        u = (t - m) * rs
        e = d * w.double() if w is not None else d
        size = e.abs() + e.abs().mean(1, keepdim=True) + u.abs() * (e * u).abs().mean(1, keepdim=True)
        return (e - (e.mean(1, keepdim=True) if kind == "layer" else 0) - u * (e * u).mean(1, keepdim=True)) * rs, size * rs * (1 + u.abs()), d * u, d

    d, size, cols = rows(dx_new), rows(dx_new).abs(), {}
    if pre != "none":
        e, s, dw, db = norm_back(rows(da), rows(x_new), st[2], st[3], get("pre", "weight"), pre)
        d, size = d + e, size + s
        cols["pre_weight"], cols["pre_bias"] = (dw, dw.abs()), (db, db.abs())
    u = rows(y) if post == "none" else (rows(y) - st[0]) * st[1]
    nn = u * (get("post", "weight").double() if get("post", "weight") is not None else 1.0) + (get("post", "bias").double() if get("post", "bias") is not None else 0.0)
    close = lambda name, t, want, size, h: None if ((rows(t) - want).abs() <= (2 * D + 32) * 2.0 ** -24 * size + h * want.abs() + 1e-30).all() else pytest.fail(name)    # noqa: E731
    close("dx", back["dx"], r * d, size, hx)
    f, fs = d * wide, size * wide.abs()
    if post != "none":
        dyv, s, dw, db = norm_back(f, rows(y), st[0], st[1], get("post", "weight"), post)
        s = s + (fs + fs.mean(1, keepdim=True) + u.abs() * (fs * u.abs()).mean(1, keepdim=True)) * st[1] * (get("post", "weight").double().abs().max() if get("post", "weight") is not None else 1.0)
        cols["post_weight"], cols["post_bias"] = (dw, fs * u.abs()), (db, fs)
    else:
        dyv, s = f, fs
    close("dy", back["dy"], dyv, s, hy)
    for key, (value, absolute) in cols.items():
        side, name = key.split("_")
        if get(side, name) is not None:
            # (the sum runs over N T rows whose elements carry up to (2 D + 32) 2^-24 of their size themselves)
            close32(key, back[key], value.sum(0), absolute.sum(0) + 0, N * T + 2 * D + 32)
            if N * T > 8 and D > 8:
                assert float((back[key].double() - value.sum(0)).norm() / value.sum(0).norm()) < 2e-5, key
        else:
            assert key not in back
    if g is not None:
        want, absolute = d * nn, size * (u.abs() * 1.6 + 0.6)
        if g.dim() == 2:
            close32("gate", back["gate"], want.view(N, T, D).sum(1), absolute.view(N, T, D).sum(1), T + 2 * D + 32)
        else:
            close32("gate", back["gate"], want.sum(0), absolute.sum(0), N * T + 2 * D + 32)


def test_first_norm_of_a_stack_and_absent_gradients():
    x = torch.randn(3, 20, 768, device="cuda")
    pre = dic.NormParams("rms", torch.rand(768, device="cuda") + 0.5, None, 1e-6)
    same, a, saved = dic.gated_norm(x, pre=pre)
    assert same is x
    scaled, a2, _ = dic.gated_norm(x, pre=pre, residual_scale=2.0, dtype=BF16)
    assert torch.equal(scaled, 2 * x) and a2.dtype == BF16
    want = norm_definition(x.double().view(60, 768), "rms", pre.weight, None, 1e-6)[0]
    assert (a.double().view(60, 768) - want).abs().max() < 1e-5
    da = torch.randn_like(a)
    both = dic.gated_norm_grad(torch.zeros_like(x), da, x, None, saved, pre=pre)
    alone = dic.gated_norm_grad(None, da, x, None, saved, pre=pre)
    assert set(alone) == {"dx", "pre_weight"} and all(torch.equal(both[k], alone[k]) for k in both)


def test_gated_norm_of_no_rows():
    x, w = torch.empty(0, 5, 96, device="cuda"), torch.ones(96, device="cuda")
    norm, gate = dic.NormParams("layer", w, w, 1e-5), torch.ones(96, device="cuda")
    x_new, a, saved = dic.gated_norm(x, x, post=norm, pre=norm, gate=gate)
    got = dic.gated_norm_grad(x_new, a, x_new, x, saved, post=norm, pre=norm, gate=gate)
    assert a.shape == x.shape and saved.shape == (4, 0) and got["dx"].shape == x.shape
    assert all(not got[k].any() and got[k].shape == (96,) for k in ("gate", "post_weight", "post_bias", "pre_weight", "pre_bias"))


def test_rows_at_any_alignment():
    """bf16 rows that start at an odd element."""
    room = torch.randn(1 + 7 * 50, device="cuda").to(BF16)
    x = room[1:].view(7, 50)
    y = torch.randn(7, 50, device="cuda").to(BF16)
    norm = dic.NormParams("layer", None, None, 1e-5)
    assert x.data_ptr() % 4 == 2
    for got, want in zip(dic.gated_norm(x, y, post=norm, pre=norm), dic.gated_norm(x.clone(), y, post=norm, pre=norm)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("D", [768, 8192])
def test_norms_of_more_than_2_31_elements(D):
    """The last rows of a tensor whose offsets pass 2^31 elements: as when they are called for alone, bit for bit."""
    rows, last = 2 ** 31 // D + 77, slice(-70, None)
    g = torch.Generator(device="cuda").manual_seed(D)
    x, y, dx_new, da = (torch.empty(1, rows, D, dtype=BF16, device="cuda").normal_(generator=g) for _ in range(4))
    norm, gate = dic.NormParams("layer", torch.rand(D, device="cuda") + 0.5, torch.rand(D, device="cuda"), 1e-5), torch.rand(D, device="cuda")
    how = dict(post=norm, pre=norm, gate=gate, residual_scale=0.9)
    x_new, a, saved = dic.gated_norm(x, y, **how)
    few = dic.gated_norm(x[:, last], y[:, last], **how)
    for got, want in zip((x_new[:, last], a[:, last], saved[:, last]), few):
        assert torch.equal(got, want)
    back = dic.gated_norm_grad(dx_new, da, x_new, y, saved, **how)
    alone = dic.gated_norm_grad(dx_new[:, last], da[:, last], few[0], y[:, last], few[2], **how)
    for name in ("dx", "dy"):
        assert torch.equal(back[name][:, last], alone[name]), name
    # a column's sum of `rows` terms in fp32, in any order: off by at most rows 2^-24 of the sum of their sizes
    d = da[0, :, -8:].double()
    assert ((back["pre_bias"][-8:].double() - d.sum(0)).abs() <= rows * 2.0 ** -24 * d.abs().sum(0)).all()


def test_sequences_of_a_cache_far_apart():
    """Sequences 5 GiB apart and heads 2.2 GiB: the results of the same rows side by side, bit for bit."""
    N, Tq, Tk, Hq, Hkv, dh = 3, 40, 100, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    q, dout = (torch.randn(N, Tq, Hq, dh, generator=g, device="cuda").to(BF16) for _ in range(2))
    k, v = (torch.randn(N, Tk, Hkv, dh, generator=g, device="cuda").to(BF16) for _ in range(2))
    step_n, step_h = 5 << 29, 9 << 27
    room = torch.empty(2 * step_n + step_h + Tk * 256, dtype=BF16, device="cuda")
    far = [room.as_strided((N, Tk, Hkv, dh), (step_n, 256, step_h, 1), 64 * i) for i in range(4)]
    far[0].copy_(k)
    far[1].copy_(v)
    for rows in (slice(0, Tq), slice(0, 2)):
        how = dict(left=30, right=0, sinks=3, q_pos=torch.tensor([60, 10, 0], dtype=torch.int32, device="cuda"))
        u, du = q[:, rows].contiguous(), dout[:, rows].contiguous()
        out, lse = dic.window_attention(u, k, v, **how)
        want = dic.window_attention_grad(du, u, k, v, out, lse, **how)
        o2, l2 = dic.window_attention(u, *far[:2], **how)
        d2 = torch.empty_like(u)
        dic.window_attention_grad(du, u, *far[:2], o2, l2, grads=(d2, far[2], far[3]), **how)
        for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *want), (o2, l2, d2, far[2], far[3])):
            assert torch.equal(a, b), name


# ------------------------------------------------------------------------------------------------ together, streams, graphs, refusals
def block(q_w, o_w, x, how, post, pre, gate, heads):
    """norm -> q|k|v Linear -> attention -> Linear -> norm, gate, residual, next norm, forward and backward, as a layer's code calls them."""
    N, T, D = x.shape
    L = dic.lib()

    def gemm(A, B, M, Nn, K, a_km, b_km):
        out = torch.empty(M, Nn, device="cuda")
        p = dic._lib.GemmParams(A=A.data_ptr(), B=B.data_ptr(), C=out.data_ptr(), M=M, N=Nn, K=K, lda=M if a_km else K, ldb=Nn if b_km else K, ldc=Nn, out_f32=1)
        dic._lib.check(L.dic_gemm(0, a_km, b_km, 0, __import__("ctypes").byref(p), torch.cuda.current_stream().cuda_stream), "gemm")
        return out

    rows = N * T
    _, a, s0 = dic.gated_norm(x, pre=pre)
    qkv = gemm(a, q_w, rows, 3 * D, D, 0, 0).view(N, T, 3, heads, D // heads)
    q, k, v = qkv.unbind(2)
    ctx, lse = dic.window_attention(q, k, v, **how)
    y = gemm(ctx, o_w, rows, D, D, 0, 0).view(N, T, D)
    x_new, b, s1 = dic.gated_norm(x, y, post=post, gate=gate, residual_scale=0.9, pre=pre)

    def backward(dx_new, db):
        g1 = dic.gated_norm_grad(dx_new, db, x_new, y, s1, post=post, gate=gate, residual_scale=0.9, pre=pre)
        dctx = gemm(g1["dy"], o_w, rows, D, D, 0, 1).view(N, T, heads, D // heads)
        dqkv = torch.empty_like(qkv)
        dic.window_attention_grad(dctx, q, k, v, ctx, lse, grads=dqkv.unbind(2), **how)
        da = gemm(dqkv, q_w, rows, D, 3 * D, 0, 1).view(N, T, D)
        g0 = dic.gated_norm_grad(g1["dx"], da, x, None, s0, pre=pre)
        d_qw, d_ow = gemm(dqkv, a, 3 * D, D, rows, 1, 1), gemm(g1["dy"], ctx, D, D, rows, 1, 1)
        return {"x": g0["dx"], "gate": g1["gate"], "q_w": d_qw, "o_w": d_ow, "pre_w": g0["pre_weight"] + g1["pre_weight"], "post_b": g1["post_bias"]}

    return x_new, b, backward


def test_a_block_of_them_together():
    N, T, D, heads = 2, 72, 768, 12
    g = torch.Generator(device="cuda").manual_seed(11)
    new = lambda *s, scale=1.0: torch.randn(*s, generator=g, device="cuda") * scale       # noqa: E731
    x, q_w, o_w, gate = new(N, T, D), new(3 * D, D, scale=0.04), new(D, D, scale=0.04), new(N, D)
    pre, post = dic.NormParams("layer", 1 + 0.1 * new(D), 0.1 * new(D), 1e-6), dic.NormParams("rms", 1 + 0.1 * new(D), 0.1 * new(D), 1e-6)
    mask = torch.ones(N, T, dtype=torch.bool, device="cuda")
    mask[1, 50:] = False
    how = dict(left=16, right=16, sinks=2, key_mask=mask)
    x_new, b, backward = block(q_w, o_w, x, how, post, pre, gate, heads)
    dx_new, db = new(N, T, D), new(N, T, D)
    got = backward(dx_new, db)

    leaves = {k: t.double().requires_grad_() for k, t in dict(x=x, q_w=q_w, o_w=o_w, gate=gate, pre_w=pre.weight, post_b=post.bias).items()}
    ln = lambda t: torch.nn.functional.layer_norm(t, (D,), leaves["pre_w"], pre.bias.double(), 1e-6)      # noqa: E731
    q, k, v = (ln(leaves["x"]) @ leaves["q_w"].T).view(N, T, 3, heads, D // heads).permute(2, 0, 3, 1, 4)
    s = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(D // heads)
    see = visible(N, T, T, 16, 16, 2, mask, None, None)
    y = torch.matmul(torch.softmax(s.masked_fill(~see[:, None], -INF), -1), v).transpose(1, 2).reshape(N, T, D) @ leaves["o_w"].T
    n = y * (y.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * post.weight.double() + leaves["post_b"]
    want_x = 0.9 * leaves["x"] + leaves["gate"][:, None] * n
    want_b = ln(want_x)
    wants = dict(zip(leaves, torch.autograd.grad((want_x * dx_new.double()).sum() + (want_b * db.double()).sum(), list(leaves.values()))))
    # six fp32 operators in a row, each good to about 1e-6 of its norm: 1e-5 leaves room for their sum
    for name, t, want in [("x_new", x_new, want_x), ("b", b, want_b)] + [(k, got[k], wants[k]) for k in got]:
        assert float((t.double() - want).norm() / want.norm()) < 1e-5, name


@pytest.mark.parametrize("T", [150, 400])
def test_captured_into_graphs_and_replayed(T):
    """Two graphs that hold both operators, forward and backward, replayed in turn with new inputs between: each replay equals the eager call."""
    N, heads, dh = 2, 4, 64
    D = heads * dh
    norm = dic.NormParams("layer", torch.rand(D, device="cuda") + 0.5, torch.rand(D, device="cuda"), 1e-6)
    gate = torch.rand(N, D, device="cuda")
    how = dict(left=33, right=0, sinks=40, kv_len=torch.tensor([T, 90], dtype=torch.int32, device="cuda"))

    def step(x, qkv, dout):
        q, k, v = qkv.unbind(2)
        out, lse = dic.window_attention(q, k, v, **how)
        few, _ = dic.window_attention(q[:, -1:], k, v, left=33, right=0, sinks=4, q_pos=torch.full((N,), T - 1, dtype=torch.int32, device="cuda"))
        x_new, a, saved = dic.gated_norm(x, out.view(N, T, D), post=norm, pre=norm, gate=gate)
        back = dic.gated_norm_grad(x_new, a, x_new, out.view(N, T, D), saved, post=norm, pre=norm, gate=gate)
        return [out, lse, few, x_new, a, *back.values(), *dic.window_attention_grad(back["dy"].view(N, T, heads, dh), q, k, v, out, lse, **how), dout + 1]

    def inputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        return [torch.randn(*s, generator=g, device="cuda").to(BF16) for s in ((N, T, D), (N, T, 3, heads, dh), (4,))]

    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        static = inputs(0)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*static)
        graphs.append((graph, static, outs))
    for turn in range(6):
        graph, static, outs = graphs[turn % 2]
        fresh = inputs(turn + 1)
        for a, b in zip(static, fresh):
            a.copy_(b)
        graph.replay()
        graphs[1 - turn % 2][0].replay()                                     # the other one behind it, with its own data
        for a, b in zip(outs, step(*fresh)):
            assert torch.equal(a, b), turn
        torch.cuda.synchronize()


def test_calls_on_two_streams_at_once():
    q = torch.randn(2, 300, 4, 64, device="cuda").to(BF16)
    want = dic.window_attention(q, q, q, left=50, right=50)
    grads = dic.window_attention_grad(q, q, q, q, *want, left=50, right=50)
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            out = dic.window_attention(q, q, q, left=50, right=50)
            got.append((*out, *dic.window_attention_grad(q, q, q, q, *out, left=50, right=50)))
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, (*want, *grads)):
            assert torch.equal(a, b)


def test_refused_arguments():
    q, k = torch.randn(2, 8, 4, 64, device="cuda"), torch.randn(2, 9, 2, 64, device="cuda")
    wide = torch.randn(2, 9, 2, 66, device="cuda")
    bad = [
        dict(q=q[0]), dict(q=q.cpu()), dict(q=q.half()), dict(k=k.to(BF16)), dict(k=k[:1]), dict(v=k[:, :8]), dict(k=k[..., :32], v=k[..., :32], q=q[..., :32]),
        dict(k=torch.randn(2, 9, 3, 64, device="cuda"), v=torch.randn(2, 9, 3, 64, device="cuda")), dict(k=wide[..., :64]), dict(k=wide[..., 1:65]),
        dict(q=q.transpose(1, 3).contiguous().transpose(1, 3)), dict(left=-1), dict(right=-2), dict(sinks=-1), dict(scale=0.0), dict(scale=math.inf), dict(scale=-1.0),
        dict(key_mask=torch.ones(2, 8, dtype=torch.bool, device="cuda")), dict(key_mask=torch.ones(2, 9, device="cuda")), dict(kv_len=torch.ones(2, dtype=torch.int64, device="cuda")),
        dict(kv_len=torch.ones(3, dtype=torch.int32, device="cuda")), dict(q_pos=torch.ones(2, dtype=torch.int32)), dict(out=q[:, :4]), dict(out=q.to(BF16)),
        dict(q=q.clone().requires_grad_()),
    ]
    for kw in bad:
        with pytest.raises((ValueError, TypeError)):
            dic.window_attention(**{**dict(q=q, k=k, v=k), **kw})
    out, lse = dic.window_attention(q, k, k)
    for kw in (dict(dout=out[:, :4]), dict(dout=out.to(BF16)), dict(lse=lse[:, :2]), dict(lse=lse.double()), dict(lse=lse.transpose(1, 2).contiguous().transpose(1, 2)), dict(out=out[:1])):
        with pytest.raises((ValueError, TypeError)):
            dic.window_attention_grad(**{**dict(dout=out, q=q, k=k, v=k, out=out, lse=lse), **kw})

    x = torch.randn(4, 6, 96, device="cuda")
    n = dic.NormParams("layer", torch.ones(96, device="cuda"))
    for kw in (dict(x=x[0, 0]), dict(x=x.cpu()), dict(x=x.half()), dict(y=x[:2]), dict(x=x.to(BF16)), dict(x=x[..., :48], y=x[..., :48]), dict(post=n._replace(kind="batch")),
               dict(post=n._replace(weight=torch.ones(95, device="cuda"))), dict(post=n._replace(weight=torch.ones(96, device="cuda", dtype=BF16))),
               dict(gate=torch.ones(95, device="cuda")), dict(gate=torch.ones(7, 96, device="cuda")), dict(gate=torch.ones(4, 96, device="cuda", dtype=BF16)), dict(y=None, post=n),
               dict(y=None), dict(dtype=BF16), dict(x=torch.zeros(2, 8200, device="cuda"), y=None, pre=dic.NormParams("rms")), dict(x=x.clone().requires_grad_())):
        with pytest.raises((ValueError, TypeError)):
            dic.gated_norm(**{**dict(x=x, y=x, post=None), **kw})
    x_new, a, saved = dic.gated_norm(x, x, pre=n)
    for kw in (dict(da=None), dict(pre=None), dict(saved=saved[:3]), dict(y=x.to(BF16)), dict(dx_new=x[:2]), dict(dx_new=None, da=None, pre=None)):
        with pytest.raises((ValueError, TypeError)):
            dic.gated_norm_grad(**{**dict(dx_new=x, da=x, x_new=x_new, y=x, saved=saved, pre=n), **kw})


class Number:
    def __float__(self):
        return 0.5


def test_numbers_that_do_not_fit_are_refused_by_name():
    """ValueError or TypeError, never another exception and never a copy to the host; whole numbers and reals of any kind are taken."""
    q = torch.randn(1, 40, 2, 64, device="cuda")
    x = torch.randn(4, 6, 96, device="cuda")
    n = dic.NormParams("layer", torch.ones(96, device="cuda"))
    on_gpu, leaf = torch.tensor(1.0, device="cuda"), torch.tensor(1.0, requires_grad=True)
    import numpy as np
    out, lse = dic.window_attention(q, q, q, scale=0.5, left=4, right=2, sinks=3)
    x_new, a, saved = dic.gated_norm(x, x, pre=n, residual_scale=0.5)
    wrong = ("0.5", b"1", None, [1.0], 1j, on_gpu, leaf, torch.ones(2), object(), 1e39, 10 ** 400, math.nan, math.inf, -math.inf)
    with torch.cuda.device(q.device):
        torch.cuda.set_sync_debug_mode("error")
        try:
            for bad in wrong:
                calls = [lambda: dic.gated_norm(x, x, pre=n, residual_scale=bad), lambda: dic.gated_norm_grad(x, a, x_new, x, saved, pre=n, residual_scale=bad),
                         lambda: dic.gated_norm(x, x, pre=n._replace(eps=bad)), lambda: dic.gated_norm_grad(x, a, x_new, x, saved, pre=n._replace(eps=bad))]
                if bad is not None:
                    for kw in (dict(scale=bad), dict(left=bad), dict(right=bad), dict(sinks=bad)):
                        if type(bad) is not int or "scale" in kw:            # (a whole number, if a large one: no bound)
                            calls += [lambda kw=kw: dic.window_attention(q, q, q, **kw), lambda kw=kw: dic.window_attention_grad(q, q, q, q, out, lse, **kw)]
                for call in calls:
                    with pytest.raises((ValueError, TypeError)):
                        call()
            for kw in (dict(left=2.5), dict(right=0.1), dict(sinks=7.5), dict(left=-0.5), dict(scale=-1), dict(scale=1e-60)):
                with pytest.raises(ValueError):
                    dic.window_attention(q, q, q, **kw)
            with pytest.raises(ValueError):
                dic.gated_norm(x, x, pre=n._replace(eps=-1e-6))
            for post in (torch.ones(96, device="cuda"), "layer", ("layer", None, None, 1e-6), n._replace(kind=[1])):
                with pytest.raises((ValueError, TypeError)):
                    dic.gated_norm(x, x, post=post)
            for half, four in ((np.float32(0.5), np.int64(4)), (torch.tensor(0.5), torch.tensor(4)), (np.float64(0.5), 4.0), (Number(), np.float32(4))):
                again = dic.window_attention(q, q, q, scale=half, left=four, right=np.int32(2), sinks=3.0)
                assert all(type(u) is torch.Tensor for u in again)
                dic.gated_norm(x, x, pre=n, residual_scale=half)
        finally:
            torch.cuda.set_sync_debug_mode("default")
    for u, v in zip(again, (out, lse)):
        assert torch.equal(u, v)
    everything, far = (dic.window_attention(q, q, q, left=b, right=b)[0] for b in (None, 10 ** 400))
    assert torch.equal(everything, far)


def test_tensors_without_memory_of_their_own_are_refused():
    q, x, n = torch.randn(3, 1, 40, 2, 64, device="cuda"), torch.randn(3, 4, 96, device="cuda"), dic.NormParams("rms")
    with pytest.raises((ValueError, TypeError)):
        torch.func.vmap(lambda t: dic.window_attention(t, t, t)[0])(q)
    with pytest.raises((ValueError, TypeError)):
        torch.func.vmap(lambda t: dic.gated_norm(t, t, pre=n)[0])(x)
    with pytest.raises((ValueError, TypeError)):
        dic.gated_norm(x[0].to_sparse(), None, pre=n)
    with pytest.raises((ValueError, TypeError)):
        dic.window_attention(q[0].to_sparse(), q[0], q[0])
    out, lse = dic.window_attention(q[0], q[0], q[0])
    with pytest.raises((ValueError, TypeError)):
        dic.window_attention_grad(out.to_sparse(), q[0], q[0], q[0], out, lse)
    with pytest.raises((ValueError, TypeError)):
        dic.window_attention(q[0, ..., :0], q[0, ..., :0], q[0, ..., :0])


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    q, x, w = torch.randn(1, 40, 2, 64, device="cuda"), torch.randn(4, 96, device="cuda"), torch.ones(96, device="cuda")
    out, lse = dic.window_attention(q, q, q)
    n = dic.NormParams("layer", w, w, 1e-5)
    how = dict(post=n, gate=w, pre=n)
    x_new, a, saved = dic.gated_norm(x, x, **how)
    fwd, bwd = dict(q=q, k=q, v=q), dict(dout=out, q=q, k=q, v=q, out=out, lse=lse)
    norm, back = dict(x=x, y=x, **how), dict(dx_new=x, da=a, x_new=x_new, y=x, saved=saved, **how)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))                 # noqa: E731
        for call, args in ((dic.window_attention, fwd), (dic.window_attention_grad, bwd), (dic.gated_norm, norm), (dic.gated_norm_grad, back)):
            call(**args)                                                     # a level without tangents is no obstacle
            for name, t in args.items():
                given = [n._replace(weight=dual(w)), n._replace(bias=dual(w))] if t is n else [dual(t)]
                for g in given:
                    with pytest.raises(ValueError, match="tangent"):
                        call(**{**args, name: g})
        with pytest.raises(ValueError, match="tangent"):
            dic.window_attention_grad(**bwd, grads=(dual(q), torch.empty_like(q), torch.empty_like(q)))
    with pytest.raises((ValueError, TypeError)):
        torch.func.jvp(lambda t: dic.gated_norm(t, x, **how)[0], (x,), (x,))
