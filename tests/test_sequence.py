"""The sequence operators (WindowScorer.attention, linear_attention, linear_attention_step, group_norm) against their
definitions in 64 bits, at the lengths, masks, strides and types where they can go wrong.

Tolerances.  u = eps/2 is half a step of a type relative to the value, U = 2^-24 that of float32.
  attention         p~ = p (1 + t): t <= u (p is rounded to the inputs' type for the second product; not for float32)
                    + E, E = 2 spread (dim + 8) U + (nk + 64) U  (the score's dot product of dim terms and its scaling,
                    exp, and sums over nk keys).  It enters the weighted sum and its normalisation: 2 (u + E) weight,
                    and the result is rounded once: u |out|.  lse: E (1 + |lse|).
  linear attention  every product of the sum once rounded to the inputs' type (the scores, or the state) and once more in
                    the sum with the others: 3 u out_abs; float32 sums and powers of the decay: E = (dim_k + 512) U, each
                    of the up to T/64 hand-overs of a state one more: (T / 64) U.  The states are float32: E state_abs.
  group norm        sums of chains of at most 16 + n / 256 additions of n values each: E = (64 + n / 256) U times the terms' size,
                    through an activation of slope <= 1.1; plus u |y|.
"""
import math
import os
import random
import sys

import pytest

torch = pytest.importorskip("torch")

from conftest import ROOT  # noqa: E402

sys.path.insert(0, ROOT)
from oracle import sequence as orc  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ALL = ["f32", "f16", "bf16"]


def half(dt):
    return torch.finfo(DT[dt]).eps / 2


@pytest.fixture(scope="module")
def sc():
    from drlvae.scorer import WindowScorer
    s = WindowScorer(0)
    yield s
    s.close()


def offs(lengths, first=0):
    o = [first]
    for n in lengths:
        o.append(o[-1] + n)
    return o


def normal(gen, shape, dt, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(DT[dt]).cuda()


def within(got, want, tol, what=""):
    got, want = got.detach().cpu().double(), want.double()
    bad_nan = torch.isnan(got) != torch.isnan(want)
    assert not bad_nan.any(), f"{what}: NaN in other places ({int(bad_nan.sum())})"
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]), what
    ok = ~(torch.isnan(want) | inf)
    over = ((got - want).abs() - tol)[ok]
    if over.numel():
        assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} over the tolerance at {int((over > 0).sum())} of {over.numel()}"


def attention_bounds(dt, q, k, v, qo, ko, **kw):
    """(out, its tolerance, lse, its tolerance) from the definition."""
    want, wl, weight, spread = orc.attention(q, k, v, qo, ko, **kw)
    nk = max([1] + [b - a for a, b in zip(ko, ko[1:])])
    E = 2 * spread * (q.shape[2] + 8) * U + (nk + 64) * U
    u = half(dt)
    return (want, 2 * ((u if dt != "f32" else 0) + E[..., None]) * weight + u * want.abs() + torch.finfo(DT[dt]).tiny,
            wl, E * (1 + torch.where(torch.isinf(wl), 0.0, wl.abs())))


def check_attention(sc, dt, q, k, v, qo, ko, layout=None, **kw):
    kw.setdefault("scale", q.shape[2] ** -0.5)
    layout = layout or sc.seq_layout(qo, None if ko is None else ko)
    out, lse = sc.attention(q, k, v, layout, return_lse=True, **kw)
    torch.cuda.synchronize()
    want, tol, wl, ltol = attention_bounds(dt, q, k, v, qo, qo if ko is None else ko, **kw)
    within(out, want, tol, "out")
    within(lse, wl, ltol, "lse")
    return out, lse


# ---- attention ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("H,G,D", [(1, 1, 8), (4, 2, 64), (6, 2, 40), (8, 1, 128), (3, 3, 16), (8, 2, 96), (70, 1, 32)])
def test_attention_packed_series(sc, dt, H, G, D):
    g = torch.Generator().manual_seed(H * 1000 + D)
    lengths = [5, 0, 130, 1, 64, 33]
    o = offs(lengths)
    q, k, v = normal(g, (o[-1], H, D), dt, 1.5), normal(g, (o[-1], G, D), dt, 1.5), normal(g, (o[-1], G, D), dt)
    check_attention(sc, dt, q, k, v, o, None)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 400])
def test_attention_lengths(sc, dt, n):
    g = torch.Generator().manual_seed(n)
    q, k, v = (normal(g, (n, h, 64), dt) for h in (2, 1, 1))
    check_attention(sc, dt, q, k, v, [0, n], None)
    check_attention(sc, dt, q, k, v, [0, n], None, causal=False)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("window", [1, 7, 25, 50, 64, 65, 200])
def test_attention_window(sc, dt, window):
    g = torch.Generator().manual_seed(window)
    o = offs([150, 0, 3, 210])
    q, k, v = (normal(g, (o[-1], h, 32), dt) for h in (4, 2, 2))
    check_attention(sc, dt, q, k, v, o, None, window=window)
    check_attention(sc, dt, q, k, v, o, None, window=window, causal=False)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 300), (3, 200), (9, 70), (40, 333), (130, 190), (5, 0), (70, 30), (200, 64)])
def test_attention_more_keys_than_rows_and_fewer(sc, dt, nq, nk):
    """Rows before the first key (nk < nq, causal) see nothing."""
    g = torch.Generator().manual_seed(nq * 7 + nk)
    qo, ko = offs([nq, 2, nq]), offs([nk, 2, 20])
    q, k, v = (normal(g, (r, h, 64), dt) for r, h in ((qo[-1], 6), (ko[-1], 2), (ko[-1], 2)))
    out, lse = check_attention(sc, dt, q, k, v, qo, ko)
    if nk < nq:
        assert torch.all(out[:nq - nk] == 0) and torch.all(lse[:nq - nk] == -math.inf)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (4, 4, 128), (32, 1, 40)])
def test_attention_step_against_a_cache(sc, dt, H, G, D):
    """One row per series; slots of 700 rows, some of them filled; lengths outside the slot are clamped to it."""
    g = torch.Generator().manual_seed(D)
    klen = [700, 1, 0, 333, 64, 65, 900, -4]
    n, cap = len(klen), 700
    q, k, v = normal(g, (n, H, D), dt), normal(g, (n * cap, G, D), dt), normal(g, (n * cap, G, D), dt)
    kl = torch.tensor(klen, dtype=torch.int32, device="cuda")
    for window in (0, 100):
        check_attention(sc, dt, q, k, v, list(range(n + 1)), [i * cap for i in range(n + 1)], k_len=kl, window=window)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("step", [False, True])
def test_attention_key_mask_and_what_lies_behind_it(sc, dt, step):
    """Masked keys hold NaN and infinities; whole series are masked; the first rows see nothing."""
    g = torch.Generator().manual_seed(3)
    ko = offs([200, 90, 64, 300])
    qo = [0, 1, 2, 3, 4] if step else ko
    q, k, v = normal(g, (qo[-1], 4, 64), dt), normal(g, (ko[-1], 2, 64), dt), normal(g, (ko[-1], 2, 64), dt)
    mask = torch.rand(ko[-1], generator=g) < 0.7
    mask[:20] = False
    mask[200:290] = False
    clean = sc.attention(q, k, v, sc.seq_layout(qo, ko), key_mask=mask.cuda(), return_lse=True)
    hole = ~mask.cuda()
    k[hole], v[hole] = float("nan"), float("inf")
    v[5] = float("nan")
    out, lse = sc.attention(q, k, v, sc.seq_layout(qo, ko), key_mask=mask.cuda(), return_lse=True)
    assert torch.equal(out, clean[0]) and torch.equal(lse, clean[1])
    k[hole], v[hole] = 0, 0
    check_attention(sc, dt, q, k, v, qo, ko, key_mask=mask.cuda())


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("what", ["v", "k", "q"])
def test_attention_values_that_are_not_finite_reach_only_the_rows_that_see_them(sc, dt, window, what):
    g = torch.Generator().manual_seed(8)
    o = offs([190, 150])
    q, k, v = (normal(g, (o[-1], h, 32), dt) for h in (4, 2, 2))
    clean, tol, clean_lse, lse_tol = attention_bounds(dt, q, k, v, o, o, scale=32 ** -0.5, window=window)
    x = {"q": q, "k": k, "v": v}[what]
    for at, value in ((70, float("nan")), (131, float("inf")), (200, float("-inf"))):
        y = x.clone()
        y[at, 0, 3] = value
        args = {"q": q, "k": k, "v": v, what: y}
        out, lse = sc.attention(args["q"], args["k"], args["v"], sc.seq_layout(o), window=window, return_lse=True)
        end = 190 if at < 190 else 340
        sees = torch.zeros(o[-1], dtype=torch.bool)
        sees[at:end if not window else min(end, at + window)] = True
        if what == "q":
            sees[:] = False
            sees[at] = True
        # the rows that do not see the value are what they are without it, each within its bound: they may have been
        # summed in another order
        within(out[~sees.cuda()], clean[~sees], tol[~sees], f"{what} {at} {value}")
        within(lse[~sees.cuda()], clean_lse[~sees], lse_tol[~sees], f"{what} {at} {value} lse")
        heads = slice(0, 2) if what != "q" else slice(0, 1)
        touched = out[sees.cuda()][:, heads]
        touched = touched[..., 3] if what == "v" else touched
        if what != "k" or math.isnan(value):       # an infinite key's score may be -inf, and then weighs nothing
            assert not torch.isfinite(touched.float()).all(-1).any() if what != "v" else not torch.isfinite(touched.float()).any()
        if what != "q":
            within(out[:, 2:], clean[:, 2:], tol[:, 2:], "the other kv head")


@pytest.mark.parametrize("dt", ALL)
def test_attention_large_scores(sc, dt):
    """Scores of some hundreds: one key takes all the weight; nothing overflows."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (normal(g, (100, 2, 64), dt, s) for s in (8.0, 8.0, 1.0))
    check_attention(sc, dt, q, k, v, [0, 100], None, scale=1.0)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("nq,nk", [(1, 30000), (150, 12000), (3, 700)])
def test_attention_one_large_score_and_a_long_flat_tail(sc, dt, nq, nk):
    """The tail's weights, exp(-17.625) = 2^-25.4 each, are below float16's smallest, but all of the result."""
    q, k = torch.zeros(nq, 2, 32), torch.zeros(nk, 1, 32)
    q[:, :, 0], k[0, 0, 0] = 17.625, 1
    v = torch.ones(nk, 1, 32)
    v[0] = 0
    q, k, v = (x.to(DT[dt]).cuda() for x in (q, k, v))
    check_attention(sc, dt, q, k, v, [0, nq], [0, nk], scale=1.0, causal=False)


@pytest.mark.parametrize("dt", ALL)
def test_attention_strides_and_layout_gaps(sc, dt):
    """Fused projections, heads before rows, rows of no series: left as they were."""
    g = torch.Generator().manual_seed(2)
    x = normal(g, (180, 4 + 2 + 2, 64), dt)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    o = [10, 100, 100, 170]
    out = torch.full((4, 180, 64), 7.0, dtype=DT[dt], device="cuda").transpose(0, 1)
    got = sc.attention(q, k.transpose(0, 1).contiguous().transpose(0, 1), v, sc.seq_layout(o), out=out)
    want = sc.attention(q.contiguous(), k.contiguous(), v.contiguous(), sc.seq_layout(o))
    assert got is out and torch.equal(out[10:170], want[10:170])
    assert torch.all(out[:10] == 7) and torch.all(out[170:] == 7) and torch.all(want[:10] == 0)
    check_attention(sc, dt, q, k, v, o, None)


def test_attention_offsets_past_32_bits(sc):
    """A cache of more than 2^32 bytes and 2^31 elements, of which the last series is asked."""
    rows, G, D = 300_000, 64, 128
    k = torch.empty(rows, G, D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 1 << 31
    g = torch.Generator().manual_seed(4)
    ko = [rows - 500, rows - 200, rows]
    k[-500:], v[-500:] = normal(g, (500, G, D), "bf16"), normal(g, (500, G, D), "bf16")
    for nq in (1, 40):
        q = normal(g, (2 * nq, G, D), "bf16")
        out, lse = sc.attention(q, k, v, sc.seq_layout([0, nq, 2 * nq], ko), return_lse=True)
        small = sc.attention(q, k[-500:], v[-500:], sc.seq_layout([0, nq, 2 * nq], [0, 300, 500]), return_lse=True)
        assert torch.equal(out, small[0]) and torch.equal(lse, small[1])


# ---- linear attention ----------------------------------------------------------------------------------------------
def log_decay(gen, H, kind="memory"):
    if kind == "memory":
        return torch.log1p(-torch.exp2(-torch.linspace(1.0, 10.0, H, dtype=torch.float64))).float().cuda()
    return torch.tensor(([0.0, -math.inf, 0.7, -0.01, -30.0] * H)[:H]).cuda()


def linear_bounds(dt, q, k, v, ld, o, scale, state=None):
    """(out, its tolerance, last states, their tolerance) from the definition."""
    want, S, oa, sa = orc.linear_attention(q, k, v, ld, o, scale=scale, state=state)
    T = max([0] + [b - a for a, b in zip(o, o[1:])])
    E = (q.shape[2] + 512 + T / 64) * U
    u = half(dt)
    return want, (3 * (u if dt != "f32" else 0) + E) * oa + u * want.abs() + torch.finfo(DT[dt]).tiny, S, E * sa + 1e-37


def check_linear(sc, dt, q, k, v, ld, o, state=None, scale=None, **kw):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out, final = sc.linear_attention(q, k, v, ld, sc.seq_layout(o), scale=scale, state=state, **kw)
    torch.cuda.synchronize()
    want, tol, S, stol = linear_bounds(dt, q, k, v, ld, o, scale, state)
    within(out, want, tol, "out")
    within(final, S, stol, "final state")
    return out, final


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("H,G,dk,dv", [(1, 1, 8, 8), (4, 2, 64, 64), (3, 3, 40, 24), (4, 1, 128, 128), (2, 2, 64, 200), (2, 1, 16, 256)])
def test_linear_packed_series(sc, dt, H, G, dk, dv):
    g = torch.Generator().manual_seed(dk * 1000 + dv)
    o = offs([70, 0, 1, 64, 200, 33])
    q, k, v = normal(g, (o[-1], H, dk), dt), normal(g, (o[-1], G, dk), dt), normal(g, (o[-1], G, dv), dt)
    check_linear(sc, dt, q, k, v, log_decay(g, H), o)
    check_linear(sc, dt, q, k, v, log_decay(g, H), o, state=normal(g, (6, H, dk, dv), "f32", 3.0))


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 700])
def test_linear_lengths(sc, dt, n):
    g = torch.Generator().manual_seed(n)
    q, k, v = (normal(g, (n, 2, 32), dt) for _ in range(3))
    check_linear(sc, dt, q, k, v, log_decay(g, 2), [0, n], state=normal(g, (1, 2, 32, 32), "f32"))


@pytest.mark.parametrize("dt", ALL)
def test_linear_decays_at_their_ends(sc, dt):
    """No decay, everything forgotten at once, a growth (taken as no decay), and a fast decay."""
    g = torch.Generator().manual_seed(6)
    o = offs([100, 150])
    q, k, v = (normal(g, (250, 5, 32), dt) for _ in range(3))
    check_linear(sc, dt, q, k, v, log_decay(g, 5, "ends"), o, state=normal(g, (2, 5, 32, 32), "f32"))


@pytest.mark.parametrize("dt", ALL)
def test_linear_a_long_series_is_cut_anywhere(sc, dt):
    """3,000 rows at once, and the same handed on from call to call; the state may be updated in place."""
    g = torch.Generator().manual_seed(9)
    q, k, v = (normal(g, (3000, 2, 64), dt) for _ in range(3))
    ld = log_decay(g, 2)
    out, final = check_linear(sc, dt, q, k, v, ld, [0, 3000])
    state = torch.zeros(1, 2, 64, 64, device="cuda")
    parts = []
    for a, b in ((0, 1), (1, 700), (700, 764), (764, 2999), (2999, 3000)):
        o, same = sc.linear_attention(q[a:b], k[a:b], v[a:b], ld, sc.seq_layout([0, b - a]), state=state, final_state=state)
        assert same is state
        parts.append(o)
    want, S, oa, sa = orc.linear_attention(q, k, v, ld, [0, 3000], scale=64 ** -0.5)
    E, u = (64 + 512 + 5 + 3000 / 64) * U, half(dt)
    within(torch.cat(parts), want, (3 * (u if dt != "f32" else 0) + E) * oa + u * want.abs(), "cut")
    within(state, S, E * sa, "cut state")


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("n,H,G,dk,dv", [(1, 1, 1, 8, 8), (5, 4, 2, 64, 64), (3, 6, 2, 40, 24), (9, 2, 2, 128, 128), (2, 2, 1, 64, 256)])
def test_linear_steps_are_the_series(sc, dt, n, H, G, dk, dv):
    g = torch.Generator().manual_seed(dk + dv)
    T = 6
    q, k, v = normal(g, (T, n, H, dk), dt), normal(g, (T, n, G, dk), dt), normal(g, (T, n, G, dv), dt)
    ld = log_decay(g, H)
    start = normal(g, (n, H, dk, dv), "f32")
    state = start.clone()
    outs = torch.stack([sc.linear_attention_step(q[t], k[t], v[t], ld, state) for t in range(T)])
    order = lambda x: x.transpose(0, 1).reshape(n * T, *x.shape[2:])  # noqa: E731
    want, S, oa, sa = orc.linear_attention(order(q), order(k), order(v), ld, [i * T for i in range(n + 1)], scale=dk ** -0.5, state=start)
    E, u = (dk + 64) * U, half(dt)
    within(order(outs), want, E * oa + u * want.abs() + torch.finfo(DT[dt]).tiny, "steps")
    within(state, S, E * sa, "state")


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("what", ["v", "k", "q"])
def test_linear_values_that_are_not_finite_reach_only_what_follows(sc, dt, what):
    g = torch.Generator().manual_seed(11)
    o = offs([150, 100])
    q, k, v = (normal(g, (250, 2, 32), dt) for _ in range(3))
    ld = log_decay(g, 2)
    clean, tol, cs, stol = linear_bounds(dt, q, k, v, ld, o, 32 ** -0.5)
    for at, value in ((75, float("nan")), (97, float("inf"))):
        y = {"q": q, "k": k, "v": v}[what].clone()
        y[at, 0, 3] = value
        args = {"q": q, "k": k, "v": v, what: y}
        out, state = sc.linear_attention(args["q"], args["k"], args["v"], ld, sc.seq_layout(o))
        # what comes before, or belongs to another series or head, is what it is without the value, each within its
        # bound: it may have been summed in another order
        free = torch.ones(250, 2, dtype=torch.bool)
        free[at:at + 1 if what == "q" else 150, 0] = False
        within(out[free.cuda()], clean[free], tol[free], f"{what} {at} {value}")
        within(state[1], cs[1], stol[1], "state of the other series")
        within(state[:, 1], cs[:, 1], stol[:, 1], "state of the other head")
        if what == "q":
            assert not torch.isfinite(out[at, 0].float()).any()
            within(state, cs, stol, "state")
        else:
            hit = state[0, 0, :, 3] if what == "v" else state[0, 0, 3]
            assert not torch.isfinite(hit).any()
            assert not torch.isfinite(out[at:150, 0, 3].float()).any()


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_linear_large_values(sc, dt):
    """Scores and states past the range of float16 where the results are inside it."""
    g = torch.Generator().manual_seed(12)
    q, k, v = normal(g, (200, 1, 128), dt, 60.0), normal(g, (200, 1, 128), dt, 60.0), normal(g, (200, 1, 32), dt, 1e-3)
    check_linear(sc, dt, q, k, v, log_decay(g, 1), [0, 200], scale=1.0)
    q, k, v = normal(g, (200, 1, 64), dt, 1e-3), normal(g, (200, 1, 64), dt, 300.0), normal(g, (200, 1, 32), dt, 300.0)
    check_linear(sc, dt, q, k, v, log_decay(g, 1), [0, 200], scale=0.5)


@pytest.mark.parametrize("dt", ALL)
def test_linear_strides_and_gaps(sc, dt):
    g = torch.Generator().manual_seed(13)
    x = normal(g, (160, 8, 64), dt)
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    o, ld = [5, 75, 75, 150], log_decay(g, 4)
    out = torch.full((160, 4, 64), 7.0, dtype=DT[dt], device="cuda")
    got, s1 = sc.linear_attention(q, k, v, ld, sc.seq_layout(o), out=out)
    want, s2 = sc.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), ld, sc.seq_layout(o))
    assert got is out and torch.equal(out[5:150], want[5:150]) and torch.equal(s1, s2)
    assert torch.all(out[:5] == 7) and torch.all(out[150:] == 7) and torch.all(s1[1] == 0)


# ---- group norm ----------------------------------------------------------------------------------------------------
def check_norm(sc, dt, x, groups, gamma, beta, o, layout, act, eps=1e-5, out=None):
    src = x.clone()
    y = sc.group_norm(x, groups, gamma, beta, layout=layout, eps=eps, activation=act, out=out)
    torch.cuda.synchronize()
    want, size = orc.group_norm(src, groups, gamma, beta, o, eps=eps, activation=act)
    n = max([1] + [b - a for a, b in zip(o, o[1:])]) * (x.shape[1] // groups)
    within(y, want, 1.1 * (64 + n / 256) * U * size + half(dt) * want.abs() + torch.finfo(DT[dt]).tiny, act)
    return y


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("C,G", [(1, 1), (3, 1), (12, 4), (32, 32), (128, 8), (130, 2), (1024, 16), (96, 3), (4096, 32), (2056, 1)])
@pytest.mark.parametrize("act", ["linear", "silu"])
def test_norm_rows(sc, dt, C, G, act):
    g = torch.Generator().manual_seed(C)
    x = normal(g, (37, C), dt, 2.0) + 1.0
    check_norm(sc, dt, x, G, normal(g, (C,), "f32"), normal(g, (C,), "f32"), list(range(38)), None, act)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("C,G", [(1, 1), (5, 5), (12, 4), (64, 8), (130, 2), (128, 1), (512, 32), (1040, 2)])
@pytest.mark.parametrize("act", ["relu", "sigmoid"])
def test_norm_series(sc, dt, C, G, act):
    g = torch.Generator().manual_seed(C + 1)
    o = offs([40, 0, 1, 333, 64], 3)
    x = normal(g, (o[-1] + 2, C), dt, 2.0) + 3.0
    y = check_norm(sc, dt, x, G, None if C == 12 else normal(g, (C,), "f32"), None if C == 64 else normal(g, (C,), "f32"), o, sc.seq_layout(o), act)
    assert torch.all(y[:3] == 0) and torch.all(y[-2:] == 0)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("rows,C,G", [(20000, 64, 4), (30000, 24, 1), (5000, 256, 1)])
def test_norm_long_series(sc, dt, rows, C, G):
    """A mean far from 0: no difference of large squares."""
    g = torch.Generator().manual_seed(rows)
    o = offs([rows, 17])
    x = (normal(g, (o[-1], C), "f32", 0.5) + 100.0).to(DT[dt])
    check_norm(sc, dt, x, G, normal(g, (C,), "f32"), normal(g, (C,), "f32"), o, sc.seq_layout(o), "silu")


@pytest.mark.parametrize("dt", ALL)
def test_norm_in_place_strided_and_constant(sc, dt):
    g = torch.Generator().manual_seed(5)
    wide = normal(g, (60, 100), dt)
    x = wide[:, 7:7 + 48]
    rest = wide.clone()
    y = check_norm(sc, dt, x, 4, None, None, list(range(61)), None, "linear", out=x)
    assert y is x and torch.equal(wide[:, :7], rest[:, :7]) and torch.equal(wide[:, 55:], rest[:, 55:])
    o = [0, 30, 60]
    x = wide[:, 10:90]
    check_norm(sc, dt, x, 2, None, None, o, sc.seq_layout(o), "silu", out=x)
    c = torch.full((9, 16), 3.0, dtype=DT[dt], device="cuda")
    beta = torch.arange(16, device="cuda", dtype=torch.float32)
    assert torch.equal(sc.group_norm(c, 4, None, beta), beta.to(DT[dt]).expand(9, 16))


@pytest.mark.parametrize("dt", ALL)
def test_norm_not_finite_stays_in_its_group(sc, dt):
    g = torch.Generator().manual_seed(6)
    x = normal(g, (50, 32), dt)
    o = [0, 20, 50]
    for layout in (None, sc.seq_layout(o)):
        clean = sc.group_norm(x, 4, layout=layout)
        y = x.clone()
        y[25, 9] = float("nan")
        got = sc.group_norm(y, 4, layout=layout)
        hit = torch.zeros(50, 32, dtype=torch.bool, device="cuda")
        hit[slice(25, 26) if layout is None else slice(20, 50), 8:16] = True
        assert torch.isnan(got[hit].float()).all() and torch.equal(got[~hit], clean[~hit])


# ---- together --------------------------------------------------------------------------------------------------------
def block(sc, x, wq, ld, gamma, beta, layout, state=None):
    """A mixer block as a network has it: fused projection, linear attention, per-head norm with SiLU, attention."""
    n = x.shape[0]
    p = (x @ wq).view(n, 8, 32)
    y, state = sc.linear_attention(p[:, :4], p[:, 4:6], p[:, 6:], ld, layout, state=state)
    y = sc.group_norm(y.reshape(n, 128), 4, gamma, beta, activation="silu").view(n, 4, 32)
    z = sc.attention(y, p[:, 4:6], p[:, 6:], layout, window=50)
    return sc.group_norm(z.reshape(n, 128), 8, gamma, beta, layout=layout, activation="relu"), state


def _block_inputs(dt):
    g = torch.Generator().manual_seed(21)
    return (normal(g, (300, 64), dt), normal(g, (64, 256), dt, 0.125), log_decay(g, 4), normal(g, (128,), "f32"), normal(g, (128,), "f32"))


@pytest.mark.parametrize("dt", ALL)
def test_a_run_of_them_together(sc, dt):
    x, w, ld, gamma, beta = _block_inputs(dt)
    o = [0, 130, 130, 131, 300]
    got, state = block(sc, x, w, ld, gamma, beta, sc.seq_layout(o))
    p = (x @ w).view(300, 8, 32)
    f = DT[dt]
    y, S, _, _ = orc.linear_attention(p[:, :4], p[:, 4:6], p[:, 6:], ld, o, scale=32 ** -0.5)
    y = orc.group_norm(y.to(f).reshape(300, 128), 4, gamma, beta, list(range(301)), eps=1e-5, activation="silu")[0].to(f).view(300, 4, 32)
    z = orc.attention(y, p[:, 4:6], p[:, 6:], o, o, scale=32 ** -0.5, window=50)[0].to(f)
    want = orc.group_norm(z.reshape(300, 128), 8, gamma, beta, o, eps=1e-5, activation="relu")[0]
    rel = float((got.cpu().double() - want).norm() / want.norm())
    assert rel < 16 * half(dt) + 1e-5, rel            # four operators, each within a few half-steps of its result
    assert float((state.cpu().double() - S).norm() / S.norm()) < 1e-5


def test_calls_are_captured_and_replayed(sc):
    """Every operator in one graph on a side stream, replayed with other inputs between eager calls; another graph of the
    same calls and layouts beside it."""
    dt = "bf16"
    g = torch.Generator().manual_seed(31)
    x, w, ld, gamma, beta = _block_inputs(dt)
    layout = sc.seq_layout([0, 130, 130, 131, 300])
    cap = 4096
    steps = sc.seq_layout([0, 1, 2], [0, cap, 2 * cap])
    kc, vc = normal(g, (2 * cap, 2, 32), dt), normal(g, (2 * cap, 2, 32), dt)
    q1 = normal(g, (2, 4, 32), dt)
    kl = torch.tensor([cap, 70], dtype=torch.int32, device="cuda")
    long = sc.seq_layout([0, 9000])
    xl = normal(g, (9000, 64), dt)
    rows = normal(g, (9000, 3, 32), dt)

    def work(xx):
        a, s = block(sc, xx, w, ld, gamma, beta, layout)
        b = sc.attention(q1, kc, vc, steps, k_len=kl)
        c = sc.linear_attention_step(q1, kc[:2], vc[:2], ld, s[:2].contiguous())
        d = sc.group_norm(xl, 4, layout=long)
        e, f = sc.linear_attention(rows[:, :1], rows[:, 1:2], rows[:, 2:], ld[:1], long)
        return a, s, b, c, d, e, f

    graphs = []
    for _ in range(2):
        xin = x.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(xin)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(xin)
        graphs.append((graph, xin, out))
    for r in range(4):
        inputs = [normal(g, (300, 64), dt) for _ in graphs]
        kl.fill_(50 + 977 * r)
        for (graph, xin, _), new in zip(graphs, inputs):
            xin.copy_(new)
        for graph, _, _ in graphs:
            graph.replay()
        want = [work(new) for new in inputs]
        torch.cuda.synchronize()
        for (_, _, out), w_ in zip(graphs, want):
            for got, exp in zip(out, w_):
                assert torch.equal(got, exp)


def test_two_streams_at_once(sc):
    dt = "bf16"
    x, w, ld, gamma, beta = _block_inputs(dt)
    layout = sc.seq_layout([0, 300])
    g = torch.Generator().manual_seed(41)
    cap = 20000
    kc, vc, q1 = normal(g, (cap, 2, 64), dt), normal(g, (cap, 2, 64), dt), normal(g, (1, 8, 64), dt)
    steps = sc.seq_layout([0, 1], [0, cap])
    want = block(sc, x, w, ld, gamma, beta, layout)[0], sc.attention(q1, kc, vc, steps)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for r in range(6):
        with torch.cuda.stream(streams[r % 3]):
            got.append((block(sc, x, w, ld, gamma, beta, layout)[0], sc.attention(q1, kc, vc, steps)))
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_the_scoring_calls_stay_usable_beside_them(sc):
    """The operators leave the context's stream and the current device as they are."""
    before = torch.cuda.current_device()
    test_a_run_of_them_together(sc, "f32")
    assert torch.cuda.current_device() == before
    sc.synchronize()


def test_empty_calls(sc):
    z = torch.empty(0, 2, 32, device="cuda")
    assert sc.attention(z, z, z, sc.seq_layout([0])).shape == (0, 2, 32)
    assert sc.attention(z, z, z, sc.seq_layout([0, 0, 0])).shape == (0, 2, 32)
    state = torch.ones(2, 2, 32, 32, device="cuda")
    out, final = sc.linear_attention(z, z, z, torch.zeros(2, device="cuda"), sc.seq_layout([0, 0, 0]), state=state)
    assert out.shape == (0, 2, 32) and torch.equal(final, state)
    out, final = sc.linear_attention(z, z, z, torch.zeros(2, device="cuda"), sc.seq_layout([0, 0, 0]))
    assert torch.all(final == 0)
    assert sc.linear_attention_step(z, z, z, torch.zeros(2, device="cuda"), torch.empty(0, 2, 32, 32, device="cuda")).shape == (0, 2, 32)
    assert sc.group_norm(torch.empty(0, 8, device="cuda"), 2).shape == (0, 8)
    q = torch.ones(3, 2, 32, device="cuda")
    out, lse = sc.attention(q, z, z, sc.seq_layout([0, 3], [0, 0]), return_lse=True)
    assert torch.all(out == 0) and torch.all(lse == -math.inf)


def test_layouts_come_and_go_under_work(sc):
    """Tables that are given back are not written over while work may read them."""
    g = torch.Generator().manual_seed(5)
    q, k, v = (normal(g, (3000, h, 64), "bf16") for h in (4, 2, 2))
    r = torch.Generator().manual_seed(6)
    kept, offsets = [], []
    for i in range(300):
        cuts = sorted(int(x) for x in torch.randint(0, 3001, (int(torch.randint(1, 90, (1,), generator=r)),), generator=r))
        offsets.append([0] + cuts + [3000])
        kept.append(sc.attention(q, k, v, sc.seq_layout(offsets[-1]), window=40))       # the layout dies with the call
    for i in range(0, 300, 7):
        layout = sc.seq_layout(offsets[i])
        assert torch.equal(sc.attention(q, k, v, layout, window=40), kept[i]), i


def test_linear_steps_of_many_series(sc):
    n, H, D = (1 << 20) - 1, 16, 8                             # 16 workgroups short of the most that one call takes
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(n, H, D, device="cuda", dtype=torch.bfloat16, generator=g) for _ in range(3))
    ld = -torch.rand(H, device="cuda", generator=g)
    state = torch.randn(n, H, D, D, device="cuda", generator=g)
    some = torch.tensor([0, 1, 77777, 524288, n - 2, n - 1], device="cuda")
    before = state[some].cpu()
    out = sc.linear_attention_step(q, k, v, ld, state, scale=0.5)
    want, final, oa, sa = orc.linear_attention(q[some], k[some], v[some], ld, list(range(len(some) + 1)), scale=0.5, state=before)
    E = (D + 512) * U
    within(out[some], want, (3 * half("bf16") + E) * oa + half("bf16") * want.abs())
    within(state[some], final, E * sa)
    with pytest.raises(Exception, match="too many"):
        sc.linear_attention_step(*(x[:1].expand(1 << 20, H, D) for x in (q, k, v)), ld, torch.empty(1 << 20, H, D, D, device="cuda"),
                                 out=torch.empty(1 << 20, H, D, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_linear_offsets_past_32_bits(sc, dt):
    n, stride = 300, 1 << 23
    big = torch.empty(n * stride, device="cuda", dtype=DT[dt])
    g = torch.Generator().manual_seed(3)
    q, k, v = (big.as_strided((n, 1, 32), (stride, 32, 1), at) for at in (0, 64, 128))
    for x in (q, k, v):
        x.copy_(normal(g, (n, 1, 32), dt))
    ld = torch.tensor([-0.1], device="cuda")
    layout = sc.seq_layout([0, n])
    out, final = sc.linear_attention(q, k, v, ld, layout)
    want, last, oa, sa = orc.linear_attention(q, k, v, ld, [0, n], scale=32 ** -0.5)
    E = (32 + 512 + n / 64) * U
    within(out, want, (3 * half(dt) + E) * oa + half(dt) * want.abs())
    within(final, last, E * sa)


@pytest.mark.parametrize("series", [False, True])
def test_norm_offsets_past_32_bits(sc, series):
    rows, C, G = 4_300_000, 512, 8                             # 2.2e9 values
    x = torch.empty(rows, C, device="cuda", dtype=torch.bfloat16).normal_()
    tail = 1000
    x[:tail] = x[-tail:]
    if series:
        y = sc.group_norm(x, G, layout=sc.seq_layout([0, tail, rows - tail, rows]), activation="silu")
    else:
        y = sc.group_norm(x, G, activation="silu")
    off = [0, tail] if series else list(range(tail + 1))
    want, size = orc.group_norm(x[-tail:], G, None, None, off, eps=1e-5, activation="silu")
    n = C // G * (tail if series else 1)
    tol = 1.1 * (64 + n / 256) * U * size + half("bf16") * want.abs()
    within(y[-tail:], want, tol)
    within(y[:tail], want, tol)


# ---- random cases, many series, the C interface ----------------------------------------------------------------------
SEEDS = int(os.environ.get("DRLVAE_SWEEP_SEEDS", 24))


def lengths_of(r, n, total):
    return [r.choice([0, 1, 2, 31, 32, 33, 64, r.randint(1, total), r.randint(1, max(1, total // 4))]) for _ in range(n)]


@pytest.mark.parametrize("seed", range(SEEDS))
def test_attention_random(sc, seed):
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    dt = r.choice(ALL)
    G = r.choice([1, 1, 2, 3])
    H, D = G * r.choice([1, 2, 3, 5, 8, 40]), 8 * r.randint(1, 16)
    n = r.randint(1, 5)
    qo = offs(lengths_of(r, n, 200 if H < 16 else 40), r.choice([0, 3]))
    ko = qo if r.random() < 0.5 else offs(lengths_of(r, n, r.choice([100, 1500])), r.choice([0, 5]))
    kr = ko[-1] + r.choice([0, 7])
    q, k, v = normal(g, (qo[-1] + r.choice([0, 2]), H, D), dt, r.choice([0.3, 1.0, 3.0])), normal(g, (kr, G, D), dt), normal(g, (kr, G, D), dt)
    mask = (torch.rand(kr, generator=g) < r.choice([0.1, 0.9])).cuda() if r.random() < 0.4 else None
    k_len = torch.tensor([r.choice([0, 1, r.randint(0, 1600), 5000]) for _ in range(n)], dtype=torch.int32, device="cuda") if r.random() < 0.4 else None
    check_attention(sc, dt, q, k, v, qo, ko, causal=r.random() < 0.7, window=r.choice([0, 0, 1, 20, 64, 300]), key_mask=mask, k_len=k_len)


@pytest.mark.parametrize("seed", range(SEEDS))
def test_linear_random(sc, seed):
    r, g = random.Random(seed + 1000), torch.Generator().manual_seed(seed)
    dt = r.choice(ALL)
    G = r.choice([1, 2, 3])
    H, dk, dv = G * r.choice([1, 2, 4]), 8 * r.randint(1, 16), 8 * r.randint(1, 32)
    n = r.randint(1, 5)
    o = offs(lengths_of(r, n, r.choice([60, 400])), r.choice([0, 3]))
    q, k, v = normal(g, (o[-1], H, dk), dt), normal(g, (o[-1], G, dk), dt), normal(g, (o[-1], G, dv), dt, r.choice([0.01, 1.0]))
    state = torch.randn(n, H, dk, dv, generator=g).cuda() if r.random() < 0.5 else None
    check_linear(sc, dt, q, k, v, log_decay(g, H, r.choice(["memory", "ends"])), o, state=state)


@pytest.mark.parametrize("seed", range(SEEDS))
def test_norm_random(sc, seed):
    r, g = random.Random(seed + 2000), torch.Generator().manual_seed(seed)
    dt = r.choice(ALL)
    G = r.choice([1, 2, 3, 8, 32])
    C = G * r.choice([1, 2, 3, 7, 8, 12, 16, 64, 130])
    n = r.randint(1, 6)
    o = offs(lengths_of(r, n, r.choice([60, 3000 if C < 600 else 100])))
    x = normal(g, (o[-1], C), dt, r.choice([0.1, 3.0])) + r.choice([0.0, 2.0])
    gamma, beta = ((torch.rand(C, generator=g) + 0.5).cuda() if r.random() < 0.7 else None for _ in range(2))
    if r.random() < 0.6:
        check_norm(sc, dt, x, G, gamma, beta, o, sc.seq_layout(o), r.choice(["linear", "relu", "sigmoid", "silu"]))
    else:
        check_norm(sc, dt, x, G, gamma, beta, list(range(len(x) + 1)), None, r.choice(["linear", "relu", "sigmoid", "silu"]))


def test_seventy_thousand_series(sc):
    n, dt = 70000, "bf16"
    g = torch.Generator().manual_seed(9)
    lengths = torch.randint(0, 4, (n,), generator=g).tolist()
    o = offs(lengths)
    q, k, v = normal(g, (o[-1], 4, 16), dt), normal(g, (o[-1], 2, 16), dt), normal(g, (o[-1], 2, 16), dt)
    ld, x = log_decay(g, 4), normal(g, (o[-1], 48), dt)
    layout = sc.seq_layout(o)
    a = sc.attention(q, k, v, layout)
    b, state = sc.linear_attention(q, k, v, ld, layout)
    c = sc.group_norm(x, 4, layout=layout)
    for s in [0, 1, n // 2, n - 2, n - 1] + torch.randint(0, n, (60,), generator=g).tolist():
        at, m = slice(o[s], o[s + 1]), [0, lengths[s]]
        want, tol, _, _ = attention_bounds(dt, q[at], k[at], v[at], m, m, scale=0.25)
        within(a[at], want, tol, s)
        want, tol, S, stol = linear_bounds(dt, q[at], k[at], v[at], ld, m, 0.25)
        within(b[at], want, tol, s)
        within(state[s:s + 1], S, stol, s)
        want, size = orc.group_norm(x[at], 4, None, None, m, eps=1e-5, activation="linear")
        within(c[at], want, 1.1 * 65 * U * size + half(dt) * want.abs(), s)


def test_the_c_interface_on_the_contexts_stream_and_its_workspaces(sc):
    """Calls without a stream run on the context's; a workspace that is too small is refused before anything is written, one
    of just the size is enough and nothing behind it is touched."""
    import ctypes as C

    from drlvae import _abi
    g = torch.Generator().manual_seed(77)
    rows, D = 6000, 64
    q, k, v = (normal(g, (rows, 2, D), "bf16") for _ in range(3))
    ld, x = log_decay(g, 2), normal(g, (rows, 64), "f32")
    layout = sc.seq_layout([0, rows])
    want = (sc.attention(q, k, v, layout), sc.linear_attention(q, k, v, ld, layout)[0], sc.group_norm(x, 1, layout=layout))
    st = (2 * D, D) * 4
    outs = [torch.full_like(w_, 7.0) for w_ in want]
    final = torch.zeros(1, 2, D, D, device="cuda")
    calls = [("attention", 2, (layout._h,), _abi.pack_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[0].data_ptr(), 0, 0, 0, *st, 2, 2, D, 1, 0, D ** -0.5)),
             ("linear_attention", 2, (layout._h,), _abi.pack_linear(q.data_ptr(), k.data_ptr(), v.data_ptr(), outs[1].data_ptr(), ld.data_ptr(), 0,
                                                                    final.data_ptr(), *st, 2, 2, D, D, D ** -0.5, 0)),
             ("group_norm", 0, (layout._h, rows), _abi.pack_norm(x.data_ptr(), outs[2].data_ptr(), 0, 0, 64, 64, 64, 1, 0, 1e-5))]
    torch.cuda.synchronize()
    for (name, code, head, args), out, exp in zip(calls, outs, want):
        def pack(ws, size):
            return _abi.pack_call(_abi.SEQ_CALL_SIZE, _abi.ABI_REVISION, code, 0, 0, ws, size)
        need = C.c_int64(0)
        assert getattr(sc._lib, f"drl_{name}_workspace")(sc._h, *head, pack(0, 0), args, C.byref(need)) == 0
        assert need.value > 0, name
        run = getattr(sc._lib, f"drl_{name}_dev")
        ws = torch.full((need.value + 256,), 0xab, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        for small in (pack(0, 0), pack(0, need.value), pack(ws.data_ptr(), need.value - 1)):
            assert run(sc._h, *head, small, args) == -1, name
        sc.synchronize()
        assert torch.all(out == 7) and torch.all(ws == 0xab), name
        assert run(sc._h, *head, pack(ws.data_ptr(), need.value), args) == 0, name
        sc.synchronize()
        assert torch.equal(out, exp), name
        assert torch.all(ws[need.value:] == 0xab), name


@pytest.mark.parametrize("dt", ALL)
def test_broadcast_rows_and_heads(sc, dt):
    """Strides of 0: one row of k for all, kv heads that share their memory, one row of q for all."""
    g = torch.Generator().manual_seed(51)
    n, D = 150, 40
    q, k, v = normal(g, (n, 4, D), dt), normal(g, (n, 1, D), dt), normal(g, (n, 1, D), dt)
    for a, b, c in ((q, k[:1].expand(n, 1, D), v), (q, k.expand(n, 2, D), v.expand(n, 2, D)), (q[:1].expand(n, 4, D), k, v[:1].expand(n, 1, D))):
        check_attention(sc, dt, a, b, c, [0, 70, n], None)
        check_linear(sc, dt, a, b, c, log_decay(g, 4), [0, 70, n])


def test_layouts_outlive_their_scorer_and_serve_others(sc):
    from drlvae.scorer import WindowScorer
    g = torch.Generator().manual_seed(52)
    q, k, v = (normal(g, (300, h, 32), "bf16") for h in (4, 2, 2))
    o = [0, 120, 300]
    other = WindowScorer(0)
    theirs = other.seq_layout(o)
    a = other.attention(q, k, v, theirs)
    other.close()
    assert torch.equal(sc.attention(q, k, v, theirs), a)
    assert torch.equal(sc.attention(q, k, v, sc.seq_layout(o)), a)
    theirs.close()
    with pytest.raises(ValueError, match="closed"):
        sc.attention(q, k, v, theirs)


def test_threads_with_streams_and_layouts_of_their_own(sc):
    import threading

    from drlvae.scorer import WindowScorer
    g = torch.Generator().manual_seed(53)
    x = [[normal(g, (2000, h, 64), "f16") for h in (4, 2, 2)] for _ in range(4)]
    ld = log_decay(g, 4)
    cuts = [[0, 13 * i + 1, 700 + i, 2000] for i in range(4)]

    def work(s, i):
        layout = s.seq_layout(cuts[i])
        a = s.attention(*x[i], layout, window=90)
        b, _ = s.linear_attention(*x[i], ld, layout)
        return a, b, s.group_norm(a.reshape(2000, 256), 4, layout=layout)

    want = [work(sc, i) for i in range(4)]
    torch.cuda.synchronize()
    bad = []

    def run(i):
        try:
            s, stream = WindowScorer(0), torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got = [work(s, i) for _ in range(40)]
            stream.synchronize()
            bad.extend((i, r) for r, outs in enumerate(got) if not all(torch.equal(u, w) for u, w in zip(outs, want[i])))
            s.close()
        except Exception as e:                                 # a thread's failure is the test's
            bad.append((i, repr(e)))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad[:3]
