"""The sequence operators where values, alignments and callers are at their ends: columns that die out, the largest values,
thousands of steps, tensors with tangents, errors that others left.  Bounds are those of test_sequence.py, with what is
added named beside it."""
import math

import pytest

torch = pytest.importorskip("torch")

from test_sequence import ALL, DT, U, half, linear_bounds, log_decay, normal, offs, within  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sc():
    from drlvae.scorer import WindowScorer
    s = WindowScorer(0)
    yield s
    s.close()


# ---- linear attention: values that die out ---------------------------------------------------------------------------
def check_linear_tiny(sc, dt, q, k, v, ld, o, state=None):
    """As check_linear; what lies below float32's normal range, 2^-126, may be taken as 0 in each of a chunk's 32 rows and
    of the dk products of a state with q.  float16: a column x of weighted values is scaled so that its largest lies in [2^13,
    2^14), and then rounded in two parts, the second one to a multiple of 2^-24: off by 2^-25, which is 2^-38 of the
    largest at most; times |k|, over a chunk's 32 rows, and for all chunks before, decayed by lam^32 < 1/2 each where only
    some rows are 0, a factor of 2 (a column of zeros loses nothing)."""
    dk = q.shape[2]
    out, final = sc.linear_attention(q, k, v, ld, sc.seq_layout(o), state=state)
    want, tol, S, stol = linear_bounds(dt, q, k, v, ld, o, dk ** -0.5, state)
    km, vm, qm = (float(x.abs().max()) for x in (k, v, q))
    floor = 2.0 ** -126 + (2 * 2.0 ** -38 if dt == "f16" else 0)
    within(final, S, stol + 32 * km * vm * floor, "final state")
    within(out, want, tol + (dk + 32 * dk * km * vm) * qm * 2.0 ** -126, "out")


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("others", [0, 63])
def test_linear_a_state_whose_columns_die_out(sc, dt, others):
    """A few columns of v hold nothing: there the first state decays through the whole range of float32.  One series alone is
    cut into pieces, one among 64 is not."""
    g = torch.Generator().manual_seed(61)
    o = offs([4200] + [1] * others)
    q, k, v = normal(g, (o[-1], 4, 16), dt), normal(g, (o[-1], 4, 16), dt), normal(g, (o[-1], 4, 32), dt)
    v[:, :, 3:7] = 0
    ld = torch.log1p(-torch.exp2(-torch.tensor([5.0, 7.0, 9.0, 12.0], dtype=torch.float64))).float().cuda()
    check_linear_tiny(sc, dt, q, k, v, ld, o, state=normal(g, (1 + others, 4, 16, 32), "f32", 3.0))


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("d", [-2.0, -2.8, -3.0, -3.5])
def test_linear_chunks_that_end_in_zeros(sc, dt, what, d):
    """In each series the rows of a chunk behind the first so many are 0 in k or v: scores and weighted values of what is
    left are powers of the decay from 1 down to nothing."""
    g = torch.Generator().manual_seed(62)
    first = [1, 2, 3, 4, 5, 6, 8, 12]
    o = offs([96] * len(first))
    q, k, v = normal(g, (o[-1], 2, 32), dt), normal(g, (o[-1], 2, 32), dt), normal(g, (o[-1], 2, 32), dt)
    x = {"k": k, "v": v}[what]
    for s, n in enumerate(first):
        for c in range(3):
            x[o[s] + 32 * c + n:o[s] + 32 * c + 32] = 0
    ld = torch.tensor([d, d - 0.1], device="cuda")
    check_linear_tiny(sc, dt, q, k, v, ld, o)
    check_linear_tiny(sc, dt, q, k, v, ld, [0, 96], state=normal(g, (1, 2, 32, 32), "f32"))


# ---- group norm: one layout, calls of several alignments -------------------------------------------------------------
@pytest.mark.parametrize("dt,C,G,lengths,widths", [("bf16", 64, 8, [8000] * 4, (80, 81)), ("f32", 128, 8, [1461] * 67, (136, 138))])
@pytest.mark.parametrize("turned", [False, True])
def test_norm_of_one_layout_at_several_alignments(sc, dt, C, G, lengths, widths, turned):
    """Column slices of parents of several widths, 16 or 32 bytes in: each call gets the scratch that it needs, whichever came
    before; the same call with a layout of its own gives the same."""
    g = torch.Generator().manual_seed(63)
    o = offs(lengths)
    layout = sc.seq_layout(o)
    for width in widths[::-1] if turned else widths:
        parent, results = normal(g, (o[-1], width), dt), [torch.zeros(o[-1], width, dtype=DT[dt], device="cuda") for _ in range(2)]
        for at in (16 // parent.element_size(), 32 // parent.element_size()):
            if at + C > width:
                continue
            x = parent[:, at:at + C]
            assert torch.equal(sc.group_norm(x, G, layout=layout), sc.group_norm(x, G, layout=sc.seq_layout(o)))
            a, b = (sc.group_norm(x, G, layout=use, out=r[:, at:at + C]) for use, r in zip((layout, sc.seq_layout(o)), results))
            assert torch.equal(a, b)


# ---- tangents ----------------------------------------------------------------------------------------------------------
def test_tensors_with_a_tangent_are_refused(sc):
    """There is no forward-mode derivative: a call must not return a result without its tangent."""
    import torch.autograd.forward_ad as fw
    x, ld = torch.randn(4, 2, 32, device="cuda"), torch.zeros(2, device="cuda")
    state, w, layout = torch.zeros(4, 2, 32, 32, device="cuda"), torch.ones(64, device="cuda"), sc.seq_layout([0, 4])
    flat = x.view(4, 64)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for i in range(3):
            a = [dual(x) if j == i else x for j in range(3)]
            for f in (lambda: sc.attention(*a, layout), lambda: sc.linear_attention(*a, ld, layout), lambda: sc.linear_attention_step(*a, ld, state)):
                with pytest.raises(ValueError, match="tangent"):
                    f()
        for f in (lambda: sc.linear_attention(x, x, x, dual(ld), layout), lambda: sc.linear_attention_step(x, x, x, ld, dual(state)),
                  lambda: sc.linear_attention(x, x, x, ld, layout, state=dual(state[:1])),
                  lambda: sc.group_norm(dual(flat), 2), lambda: sc.group_norm(flat, 2, dual(w)), lambda: sc.group_norm(flat, 2, w, dual(w)),
                  lambda: sc.attention(x, x, x, layout, out=dual(x))):
            with pytest.raises(ValueError, match="tangent"):
                f()
        want = sc.attention(x, x, x, layout)                     # a tensor without one is none the worse
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda t: sc.group_norm(t, 2), (flat,), (flat,))
    assert torch.equal(sc.attention(x, x, x, layout), want)


# ---- errors that others left -------------------------------------------------------------------------------------------
def test_an_error_that_someone_else_left_is_not_taken_for_the_calls_own(sc):
    """The runtime keeps the last error of a thread until it is asked for: a call that went well neither reports it nor clears it."""
    import ctypes as C
    with open("/proc/self/maps") as f:
        hip = C.CDLL({line.split()[-1] for line in f if "libamdhip64" in line}.pop())
    g = torch.Generator().manual_seed(64)
    q, state, ld = normal(g, (3, 2, 32), "f32"), torch.zeros(3, 2, 32, 32, device="cuda"), log_decay(g, 2)
    out, y = torch.empty_like(q), torch.empty(3, 64, device="cuda")
    calls = [lambda: sc.linear_attention_step(q, q, q, ld, state, out=out), lambda: sc.group_norm(q.view(3, 64), 2, out=y)]
    for call in calls:
        call()
        hip.hipGetLastError()
        left = hip.hipSetDevice(1 << 20)                         # no such device: the runtime says so, nothing else happens
        assert left != 0
        try:
            call()
        finally:
            kept = hip.hipGetLastError()
        assert kept == left
        assert hip.hipGetLastError() == 0


# ---- linear attention: thousands of steps ------------------------------------------------------------------------------
def test_linear_steps_decay_as_much_as_the_series_do(sc):
    """2,000 steps of nothing new: exp(d) must not be off by the same amount in each.  A step rounds the state once, by at most
    U and to either side: the mean over 16,384 elements is sqrt(2000 / (3 x 16384)) U = 0.2 U off, 10 U at the very most; the
    rate itself is known to 2 U of d a step."""
    d = torch.tensor([-1e-3, -3.3e-4, -0.0101, -7e-5, 0.0, -0.0], device="cuda")
    g = torch.Generator().manual_seed(65)
    start = (1 + torch.rand(1, 6, 128, 128, generator=g)).cuda()
    state, N = start.clone(), 2000
    zero = torch.zeros(1, 6, 128, device="cuda")
    for _ in range(N):
        sc.linear_attention_step(zero, zero, zero, d, state)
    want = torch.exp(d.double() * N)
    off = ((state.double() / start.double()).mean((0, 2, 3)) / want - 1).abs()
    assert torch.all(off <= 10 * U + 2 * U * N * d.double().abs()), off
    assert torch.equal(state[:, 4:], start[:, 4:])
    # a state that is not finite: as it was, decayed
    state[0, :, 0, 0], state[0, :, 0, 1] = math.inf, math.nan
    sc.linear_attention_step(zero, zero, zero, d, state)
    assert torch.all(state[0, :, 0, 0] == math.inf) and torch.isnan(state[0, :, 0, 1]).all() and torch.isfinite(state[0, :, 1:]).all()


# ---- attention: the largest values of a type ---------------------------------------------------------------------------
@pytest.mark.parametrize("nq,nk", [(64, 400), (64, 3000), (1, 400), (1, 30000)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_float16s_largest_values_stays_finite(sc, nq, nk, sign):
    """A mean of values of 65504 is 65504; the weights here are all rounded up, by 3.5e-4, which would carry it past the type's
    range.  A column that holds an infinity does not get a finite value."""
    z = math.log(64.04 / 128)
    hi = torch.tensor(z).half()
    q, k, v = (torch.zeros(n, 1, 32, dtype=torch.float16) for n in (nq, nk, nk))
    q[:, :, :2] = 1
    k[1:, :, 0], k[1:, :, 1] = hi, (z - hi.double()).half()
    v[:] = sign * 65504.0
    v[:, :, 5] = 0
    v[nk // 2, :, 5] = sign * math.inf
    out = sc.attention(q.cuda(), k.cuda(), v.cuda(), sc.seq_layout([0, nq], [0, nk]), scale=1.0, causal=False)
    keep = [d for d in range(32) if d != 5]
    assert not torch.isfinite(out[..., 5]).any()
    assert torch.isfinite(out[..., keep]).all()
    assert float((out[..., keep].double().cpu() - sign * 65504.0).abs().max()) <= 65504 * 3 * half("f16")


# ---- group norm: the activations' far ends ------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
@pytest.mark.parametrize("rows,G,series", [(5, 16, False), (5, 1, False), (40, 16, True), (40, 1, True)])
def test_norm_activations_keep_their_relative_error(sc, act, rows, G, series):
    """gamma 0: y = act(beta), at beta from -80 to 80.  exp by a base of 2 within 2 U (its argument in two parts, the second
    one's own rounding far below U), a sum U, a reciprocal 2 U, a product U; 2 U for what second orders there are: 8 U.  At
    -200 the result, 1e-87, is none of float32's: 2^-126, where its normal range ends."""
    beta = torch.linspace(-80, 80, 4096)
    beta[7::512] = torch.tensor([math.inf, -math.inf, math.nan, 1e30, -1e30, 200.0, -200.0, 3e38])
    g = torch.Generator().manual_seed(66)
    x = normal(g, (rows, 4096), "f32")
    y = sc.group_norm(x, G, torch.zeros(4096, device="cuda"), beta.cuda(), layout=sc.seq_layout([0, rows]) if series else None, activation=act)
    b = beta.double()
    want = (torch.sigmoid(b) if act == "sigmoid" else b * torch.sigmoid(b)).expand(rows, 4096)
    within(y, want, 8 * U * want.abs() + 2.0 ** -126, act)


# ---- arguments that are something else -----------------------------------------------------------------------------------
def test_arguments_of_another_kind_are_refused_by_name(sc):
    x, ld, layout = torch.zeros(4, 2, 32, device="cuda"), torch.zeros(2, device="cuda"), sc.seq_layout([0, 4])
    none = torch.zeros(4, 2, 0, device="cuda")
    for f, match in ((lambda: sc.attention(x, x, x, layout, key_mask=[True] * 4), "key_mask"), (lambda: sc.attention(x, x, x, layout, k_len=[4]), "k_len"),
                     (lambda: sc.attention(x, x, x, layout, scale=1e300), "scale"), (lambda: sc.linear_attention(x, x, x, ld, layout, scale=1e300), "scale"),
                     (lambda: sc.linear_attention_step(x, x, x, ld, torch.zeros(4, 2, 32, 32, device="cuda"), scale=-1e39), "scale"),
                     (lambda: sc.group_norm(x.view(4, 64), 2, eps=1e300), "eps"), (lambda: sc.group_norm(x.view(4, 64), 1 << 40), "groups"),
                     (lambda: sc.attention(none, none, none, layout), "dim"), (lambda: sc.linear_attention(none, none, x, ld, layout), "dim"),
                     (lambda: sc.linear_attention_step(none, none, x, ld, torch.zeros(4, 2, 0, 32, device="cuda")), "dim")):
        with pytest.raises((ValueError, RuntimeError), match=match):
            f()


# ---- attention: runs of keys ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("nq,nk", [(1, 400), (1, 700), (9, 1500), (64, 1500)])
def test_attention_joins_runs_of_keys_by_what_they_hold(sc, dt, nq, nk):
    """Scores of 1.875 x 2^18 that float32 holds exactly, of a few keys, and others far below: the mean of the tied keys' values, to
    the roundings of the weights, the sum and the result.  A log-sum of 491,520 is itself rounded to 1/32, which would weigh runs that hold
    one and three of the keys alike to 3 %."""
    g = torch.Generator().manual_seed(69)
    a, b = 1.25 * 2.0 ** 7, 1.5 * 2.0 ** 6
    q, k, v = torch.full((nq, 1, 32), a), torch.full((nk, 1, 32), b / 4), normal(g, (nk, 1, 32), dt)
    at = torch.tensor([0, 1, 2, nk - 1])                      # three in the first run, one in the last
    k[at] = b
    out = sc.attention(q.to(DT[dt]).cuda(), k.to(DT[dt]).cuda(), v, sc.seq_layout([0, nq], [0, nk]), scale=1.0, causal=False)
    want = v[at.cuda()].double().cpu().mean(0).expand(nq, 1, 32)
    size = v[at.cuda()].double().cpu().abs().mean(0).expand(nq, 1, 32)
    within(out, want, half(dt) * (want.abs() + size) + (nk + 64) * U * size, "ties")


# ---- attention: enormous scores ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("nq,nk", [(64, 400), (64, 3000), (1, 400), (1, 30000), (3, 700)])
@pytest.mark.parametrize("std", [300.0, 3000.0, 16000.0])
def test_attention_of_enormous_scores_stays_a_mean(sc, dt, nq, nk, std):
    """float32 says nothing about which key wins where scores of 1e6 to 1e11 are closer than their roundings; but the result is a
    mean of the values, 1 where these are all 1 (rounded weights: 2 u), and the log-sum is near the largest score: the
    dot product's 64 roundings of U, and one each for scale, product with log2 e and back."""
    g = torch.Generator().manual_seed(67)
    q, k, v = ((torch.randn(n, 2, 64, generator=g) * s).clamp(-60000, 60000).to(DT[dt]).cuda() for n, s in ((nq, std), (nk, std), (nk, 1.0)))
    v[..., :8] = 1
    for kw in ({}, {"key_mask": (torch.rand(nk, generator=g) < 0.5).cuda()}):
        out, lse = sc.attention(q, k, v, sc.seq_layout([0, nq], [0, nk]), scale=0.125, causal=False, return_lse=True, **kw)
        z = torch.einsum("ihd,jhd->ihj", q.double().cpu(), k.double().cpu()) * 0.125
        size = torch.einsum("ihd,jhd->ihj", q.double().cpu().abs(), k.double().cpu().abs()) * 0.125
        if kw:
            z[..., ~kw["key_mask"].cpu()] = -math.inf
        want = torch.logsumexp(z, 2)
        within(out[..., :8], torch.ones(nq, 2, 8), 3 * half(dt) + (nk + 64) * U, "mean of ones")
        within(lse, want, (64 + 8) * U * size.amax(2) + math.log(nk), "lse")
        assert float(out.abs().max()) <= float(v.abs().max()) * (1 + 3 * half(dt) + 1e-5)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("nq,nk,ties", [(64, 400, 5), (64, 3000, 7), (1, 400, 5), (1, 30000, 300), (3, 200, 7), (9, 30000, 1)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_enormous_scores_that_are_exact(sc, dt, nq, nk, ties, sign):
    """Scores of 1.875 x 2^33 that float32 holds exactly, and others far below, or far below 0: the mean of the tied keys' values,
    to the roundings of the sum and of the result."""
    g = torch.Generator().manual_seed(68)
    a, b = 1.25 * 2.0 ** 14, 1.5 * 2.0 ** 14
    q, k, v = torch.full((nq, 1, 32), a), torch.full((nk, 1, 32), b if sign < 0 else b * (1 - 2.0 ** -6)), normal(g, (nk, 1, 32), dt)
    at = torch.randperm(nk, generator=g)[:ties]
    k[::3] /= 4
    if sign < 0:
        k *= -2
    k[at] = -b / 4 if sign < 0 else b
    at = at if sign > 0 else (k[:, 0, 0] == k.max()).nonzero()[:, 0]
    out = sc.attention(q.to(DT[dt]).cuda(), k.to(DT[dt]).cuda(), v, sc.seq_layout([0, nq], [0, nk]), scale=1.0, causal=False)
    want = v[at.cuda()].double().cpu().mean(0).expand(nq, 1, 32)
    size = v[at.cuda()].double().cpu().abs().mean(0).expand(nq, 1, 32)
    within(out, want, half(dt) * want.abs() + (nk + 64) * U * size, "ties")


@pytest.mark.parametrize("seed", range(36))
def test_attention_random_cases_of_scores_that_are_exact(sc, seed):
    """Whole numbers times 2^e: every score is exact in float32, and scores that are not tied differ by 4^e, 64 at least: each row
    is the mean of its largest keys' values, whatever the lengths, masks, windows and runs."""
    import random

    from oracle import sequence as orc
    from test_sequence import lengths_of
    r, g = random.Random(seed), torch.Generator().manual_seed(seed)
    dt = ALL[seed % 3]
    G, D = r.choice([1, 2]), 8 * r.randint(1, 16)
    H = G * r.choice([1, 2, 5, 8])
    n = r.randint(1, 4)
    qo = offs(lengths_of(r, n, r.choice([3, 200])))
    ko = qo if r.random() < 0.4 else offs(lengths_of(r, n, r.choice([100, 2500])))
    e = r.choice([3, 7, 10, 12])
    whole = lambda rows, heads: (torch.randint(-3, 4, (rows, heads, D), generator=g) * 2.0 ** e).to(DT[dt]).cuda()  # noqa: E731
    q, k, v = whole(qo[-1], H), whole(ko[-1], G), normal(g, (ko[-1], G, D), dt)
    if r.random() < 0.3:
        q, k = q.abs(), -k.abs()                                # all scores below 0
    mask = (torch.rand(ko[-1], generator=g) < r.choice([0.2, 0.9])).cuda() if r.random() < 0.5 else None
    kw = dict(scale=1.0, causal=r.random() < 0.6, window=r.choice([0, 0, 7, 64, 300]), key_mask=mask)
    out, lse = sc.attention(q, k, v, sc.seq_layout(qo, ko), return_lse=True, **kw)
    want, wl, weight, _ = orc.attention(q, k, v, qo, ko, **kw)
    nk = max([1] + [b - a for a, b in zip(ko, ko[1:])])
    # references past 2^10 are rounded, by U times themselves, which all weights of a row share; two tiles' differ by that
    top = torch.where(torch.isinf(wl), 0.0, wl.abs())
    E = (nk + 64) * U + torch.where(top * 1.45 > 2.0 ** 20, 0.0, 4 * U * top)
    within(out, want, (half(dt) + E[..., None]) * weight + half(dt) * want.abs() + torch.finfo(DT[dt]).tiny, "out")
    within(lse, wl, 4 * U * top + (nk + 64) * U + torch.where(top > 2.0 ** 20, math.log(nk) + 5, 0.0), "lse")


# ---- linear attention: silence ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("others", [0, 63])
@pytest.mark.parametrize("silent", [24, 64, 107])
def test_linear_states_keep_their_relative_error_in_silence(sc, dt, others, silent):
    """40 rows and then nothing: what is left of the state, 1e-2 to 1e-19 of it, is off by its own roundings, not by those of what
    it was.  float16: the last rows' chunk loses 2^-38 of its largest weighted value (times k, 32 rows), which decays as the
    state does."""
    g = torch.Generator().manual_seed(70)
    o = offs([40 + silent] + [1] * others)
    q, k, v = normal(g, (o[-1], 4, 32), dt), normal(g, (o[-1], 4, 32), dt), normal(g, (o[-1], 4, 64), dt)
    for x in (k, v):
        x[40:40 + silent] = 0
    ld = torch.tensor([-0.02, -0.1, -0.2, -0.4], device="cuda")
    state = normal(g, (1 + others, 4, 32, 64), "f32", 3.0)
    out, final = sc.linear_attention(q, k, v, ld, sc.seq_layout(o), state=state)
    want, tol, S, stol = linear_bounds(dt, q, k, v, ld, o, 32 ** -0.5, state)
    left = torch.exp(ld.double().cpu() * silent)[None, :, None, None]
    floor = 32 * float(k.abs().max()) * float(v.abs().max()) * 2.0 ** -38 if dt == "f16" else 0.0
    within(final, S, stol + floor * left, "final state")
    within(out, want, tol, "out")


def test_linear_steps_keep_their_relative_error_in_silence(sc):
    """A state alone for 12 steps at rates from -1e-4 to -6: each step rounds twice at most, and knows exp(d) to 4 U and 2 U of |d|."""
    d = torch.tensor([-1e-4, -0.1, -0.5, -0.69, -0.7, -2.0, -6.0, -math.inf], device="cuda")
    g = torch.Generator().manual_seed(71)
    start = (1 + torch.rand(1, 8, 32, 32, generator=g)).cuda()
    state, zero, N = start.clone(), torch.zeros(1, 8, 32, device="cuda"), 12
    for _ in range(N):
        sc.linear_attention_step(zero, zero, zero, d, state)
    want = start.double() * torch.exp(d.double() * N)[None, :, None, None]
    within(state, want.cpu(), want.cpu() * (N * 2 * U * (3 + d[:7].abs().max().item())), "state")


def test_linear_states_of_a_long_series_do_not_drift(sc):
    """100,000 rows of which only the first holds anything, at memories of 20,000 rows to ever: lam^32, rounded, is off by up to 2^-25
    in each of 3,125 chunks (one series among many) or lam^n in each of a few hundred pieces: together less than 2^-22 and the
    states' own roundings, U each to either side: 8 sqrt(3125) U at the very most over their mean, 2 U of the rate."""
    T = 100_000
    d = torch.tensor([-5e-5, -1.7e-5, -3.1e-6, 0.0], device="cuda")
    for dt in ("f32", "bf16"):
        for others in (0, 63):
            o = offs([T] + [1] * others)
            q, k, v = (torch.zeros(o[-1], 4, 32, dtype=DT[dt], device="cuda") for _ in range(3))
            g = torch.Generator().manual_seed(72)
            state = (1 + torch.rand(1 + others, 4, 32, 32, generator=g)).cuda()
            _, final = sc.linear_attention(q, k, v, d, sc.seq_layout(o), state=state)
            want = torch.exp(d.double() * T)
            off = ((final[0].double() / state[0].double()).mean((1, 2)) / want - 1).abs()
            assert torch.all(off <= 4 * U + 8 * math.sqrt(3125 / 3 / 1024) * U + 2 * U * T * d.double().abs()), (dt, others, off)


@pytest.mark.parametrize("rows", [32, 50])
def test_linear_states_that_are_handed_on_do_not_drift(sc, rows):
    """3,000 calls of a chunk or two that hold nothing new: a call must not take the same rounding of lam^n each time.  Per call
    and column the factor is off by at most U to either side, the state's rounding by U: 8 sqrt(3000 / 3 / 32) U at the
    very most over the mean of 32 columns, 2 U of the rate."""
    N = 3000
    d = torch.tensor([-1e-4, -3.3e-5, -7.1e-6, -2e-4], device="cuda")          # at most e^-30: float32's normal range
    for dt, others in (("f32", 0), ("bf16", 0), ("f16", 63)):
        o = offs([rows] + [1] * others)
        layout = sc.seq_layout(o)
        q, k, v = (torch.zeros(o[-1], 4, 32, dtype=DT[dt], device="cuda") for _ in range(3))
        g = torch.Generator().manual_seed(73)
        state = (1 + torch.rand(1 + others, 4, 32, 32, generator=g)).cuda()
        start = state.clone()
        for _ in range(N):
            sc.linear_attention(q, k, v, d, layout, state=state, final_state=state)
        want = torch.exp(d.double() * (N * rows))
        off = ((state[0].double() / start[0].double()).mean((1, 2)) / want - 1).abs()
        assert torch.all(off <= 8 * math.sqrt(N / 3 / 32) * U + 2 * U * N * rows * d.double().abs()), (dt, off)
