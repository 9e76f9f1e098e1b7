"""The operators around the routed experts on the GPU against plain definitions in 64 bits.

Tolerances come from counting roundings: u = 2^-24 (half a step of fp32) for every fp32
operation, and half a step of the output's type for the last one.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ("float32", "bfloat16", "float16")
TINY = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}  # half the least subnormal


@pytest.fixture(scope="module")
def cb(cuda):
    import crosslane_b200
    return crosslane_b200


def half_step(torch, name):
    return torch.finfo(getattr(torch, name)).eps / 2


def pitched(torch, values, dtype, pad):
    """values [T][W] in rows of a buffer that is `pad` elements wider, the rest a canary."""
    t = torch.full((values.shape[0], values.shape[1] + pad), 7.0, dtype=dtype, device="cuda")
    v = t[:, : values.shape[1]]
    v.copy_(torch.as_tensor(values))
    return v


# ---------------------------------------------------------------------------- routing

def scores64(kind, l):
    there = ~np.isneginf(l)
    low = np.where(there, l, 0.0)
    with np.errstate(over="ignore"):
        if kind == "sigmoid":
            return 1.0 / (1.0 + np.exp(-low))
        if kind == "sqrt_softplus":
            return np.sqrt(np.maximum(low, 0.0) + np.log1p(np.exp(-np.abs(low))))
    top = np.where(there, l, -np.inf).max()
    if np.isneginf(top):
        return np.zeros_like(l)
    e = np.where(there, np.exp(np.where(there, l - top, 0.0)), 0.0)
    return e / e.sum()


def route64(l32, bias, k, kind, groups, top_groups, pair, renorm, scale):
    """One row by the definition: (ids, weights, is the row bad)."""
    E = l32.size
    if not np.all(l32 < np.inf) or (bias is not None and not np.all(bias < np.inf)):
        return np.arange(k), np.full(k, np.nan), True
    s = scores64(kind, l32.astype(np.float64))
    held = s.astype(np.float32)
    there = ~np.isneginf(l32) if bias is None else ~(np.isneginf(l32) | np.isneginf(bias))
    ninf = np.float32(-np.inf)
    with_bias = held if bias is None else held + bias
    rank = np.where(there, l32 if bias is None else with_bias, ninf)
    if groups > 1:
        per = E // groups
        value = np.empty(groups, np.float32)
        for g in range(groups):
            own = np.sort(np.where(there, with_bias, ninf)[g * per:(g + 1) * per])[::-1]
            if pair:
                value[g] = own[0] if per == 1 or np.isneginf(own[1]) else own[0] + own[1]
            else:
                value[g] = rank[g * per:(g + 1) * per].max()
        for g in np.argsort(-value, kind="stable")[top_groups:]:
            rank[g * per:(g + 1) * per] = ninf
    ids = np.argsort(-rank, kind="stable")[:k]
    w = np.where(np.isneginf(rank[ids]), 0.0, s[ids])
    if renorm:
        w = w / (w.sum() + 1e-20)
    return ids, w * scale, False


def check_route(torch, op, logits, bias, ids, w, kind, groups=1, top_groups=1, pair=True, renorm=True, scale=1.0):
    k = op.k
    l32 = logits.float().cpu().numpy()
    b = None if bias is None else bias.cpu().numpy()
    gi, gw = ids.cpu().numpy(), w.cpu().numpy().astype(np.float64)
    bad_rows = 0
    for t in range(l32.shape[0]):
        wi, ww, bad = route64(l32[t], b, k, kind, groups, top_groups, pair, renorm, scale)
        bad_rows += bad
        assert np.array_equal(gi[t], wi), (t, gi[t], wi)
        if bad:
            assert np.all(np.isnan(gw[t])), t
            continue
        # A score: expf and log1pf within 2 ulp (4 u each), a division within 2 ulp (4 u), additions
        # and the root 1 u each: 9 u. Softmax: an exponential of 6 u over a sum; a term exp(d) of
        # the sum is off by |d| u in its argument and 4 + 2.4 |d| u in __expf, and the mean of |d|
        # weighted by the terms is the entropy less the top's own, at most ln E <= 7; 37 additions
        # in a chain (32 of a lane, 5 of the tree): 4 + 3.4 * 7 + 37 = 65 u; the division: 75 u.
        # Renormalised: the same again for the picks' sum, with its k additions, 1e-20 and the
        # division. Then the scale. Scores below 2^-126 may be flushed.
        sc = 75 if kind == "softmax" else 9
        tol = (2 * sc + k + 4 if renorm else sc + 2) * U * np.abs(ww) + 2.0 ** -149 * max(1.0, scale)
        s = np.where(ww > 0, scores64(kind, l32[t].astype(np.float64))[wi], 0.0)
        tol += 2.0 ** -125 * scale / ((s.sum() + 1e-20) if renorm else 1.0)
        assert np.all(np.abs(gw[t] - ww) <= tol), (t, gw[t], ww)
    return bad_rows


@pytest.mark.parametrize("kind", ["sigmoid", "softmax", "sqrt_softplus"])
@pytest.mark.parametrize("E,k,groups,top,pair", [(1, 1, 1, 1, True), (2, 2, 1, 1, True), (31, 16, 1, 1, True),
                                                 (100, 6, 1, 1, True), (128, 8, 1, 1, True), (384, 6, 1, 1, True),
                                                 (384, 8, 8, 4, True), (384, 8, 8, 4, False), (256, 8, 32, 3, True),
                                                 (96, 5, 3, 2, True), (32, 3, 32, 3, True), (352, 7, 11, 2, False),
                                                 (1024, 16, 1, 1, True), (1000, 16, 4, 1, True)])
@pytest.mark.parametrize("with_bias", [False, True])
def test_route_matches_definition(cb, cuda, kind, E, k, groups, top, pair, with_bias):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(E * 31 + k)
    T = 67
    logits = torch.randn((T, E), generator=gen, device="cuda") * 3
    if E > 8:  # masked experts, ties, extremes, a row with few experts, an empty row
        logits[1::5] = torch.where(torch.rand((len(range(1, T, 5)), E), generator=gen, device="cuda") < 0.4, -math.inf,
                                   logits[1::5])
        logits[2] = 0.25
        logits[3, ::2] = 1.0
        logits[4] = torch.linspace(-120, 120, E, device="cuda")
        logits[5] = -math.inf
        logits[6] = -math.inf
        logits[6, E - 2] = -2.0
        logits[7] = torch.finfo(torch.float32).min
        logits[7, 4] = 0.0
        logits[8, ::3] = -0.0
        logits[8, 1::3] = 0.0
    bias = torch.randn(E, generator=gen, device="cuda") * 0.3 if with_bias else None
    if with_bias and E > 8:
        bias[5] = -math.inf
    op = cb.ExpertRoute(E, k, score=kind, n_groups=groups, top_groups=top, group_score="pair" if pair else "max",
                        renormalize=E % 3 != 1, scale=2.5)
    ids = torch.full((T, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), -7.0, device="cuda")
    op.run(logits, ids, w, d_bias=bias)
    assert check_route(torch, op, logits, bias, ids, w, kind, groups, top, pair, E % 3 != 1, 2.5) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pad", [0, 1, 8])
def test_route_types_and_pitches(cb, cuda, dtype, pad):
    torch = cuda
    T, E, k = 130, 384, 6
    gen = torch.Generator(device="cuda").manual_seed(7)
    logits = pitched(torch, torch.randn((T, E), generator=gen, device="cuda") * 2, getattr(torch, dtype), pad)
    bias = torch.randn(E, generator=gen, device="cuda") * 0.1
    op = cb.ExpertRoute(E, k, scale=1.5)
    back = torch.full((T + 2, k), -7, dtype=torch.int32, device="cuda")
    wback = torch.full((T + 2, k), -7.0, device="cuda")
    op.run(logits, back[:T], wback[:T], d_bias=bias)
    check_route(torch, op, logits, bias, back[:T], wback[:T], "sigmoid", scale=1.5)
    assert bool((back[T:] == -7).all()) and bool((wback[T:] == -7).all())  # rows behind the last stay


@pytest.mark.parametrize("T", [0, 1, 2, 5, 4099])
def test_route_token_counts(cb, cuda, T):
    torch = cuda
    E, k = 48, 4
    logits = torch.randn((T, E), generator=torch.Generator(device="cuda").manual_seed(T), device="cuda")
    ids = torch.empty((T, k), dtype=torch.int32, device="cuda")
    w = torch.empty((T, k), device="cuda")
    op = cb.ExpertRoute(E, k, score="softmax", renormalize=False)
    op.run(logits, ids, w)
    check_route(torch, op, logits, None, ids, w, "softmax", renorm=False)


@pytest.mark.parametrize("with_bias", [False, True])
def test_route_flags_bad_rows_alone(cb, cuda, with_bias):
    torch = cuda
    T, E, k = 9, 384, 6
    logits = torch.randn((T, E), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    logits[2, 17] = math.nan
    logits[4, 383] = math.inf
    bias = torch.zeros(E, device="cuda") if with_bias else None
    ids = torch.empty((T, k), dtype=torch.int32, device="cuda")
    w = torch.empty((T, k), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    op = cb.ExpertRoute(E, k)
    op.run(logits, ids, w, d_bias=bias, d_status=status)
    assert check_route(torch, op, logits, bias, ids, w, "sigmoid") == 2 and int(status) == 1
    status.zero_()
    op.run(logits[5:], ids[5:], w[5:], d_bias=bias, d_status=status)
    assert int(status) == 0
    if with_bias:
        bias[3] = math.nan
        op.run(logits, ids, w, d_bias=bias, d_status=status)
        assert int(status) == 1 and bool(torch.isnan(w).all()) and bool((ids == torch.arange(k, device="cuda")).all())


def close_bias(kind, l, chosen, rng, target=0.9):
    """A bias that puts the ranks of `chosen` within a few ulps of one another, above the others'."""
    held = scores64(kind, l.astype(np.float64)).astype(np.float32)
    bias = (rng.standard_normal(l.size) * 0.01 - 3.0).astype(np.float32)
    top = np.float32(target + held.max())
    bias[chosen] = top - held[chosen]
    bias[chosen] += (rng.integers(-2, 3, len(chosen)) * np.spacing(top)).astype(np.float32)
    return bias


@pytest.mark.parametrize("kind", ["sigmoid", "softmax", "sqrt_softplus"])
@pytest.mark.parametrize("E,k,near", [(384, 6, 10), (384, 8, 31), (384, 8, 384), (64, 16, 64), (256, 8, 60), (1000, 1, 2)])
def test_route_ranks_an_ulp_apart(cb, cuda, kind, E, k, near):
    """Ranks closer than fp32 scores can tell: a few candidates, and more than a warp has lanes."""
    torch = cuda
    for seed in range(6):
        rng = np.random.default_rng(seed * 1000 + E + near)
        l = (rng.standard_normal((3, E)) * 2).astype(np.float32)
        bias = close_bias(kind, l[0], rng.permutation(E)[:near], rng)
        logits, b = torch.from_numpy(l).cuda(), torch.from_numpy(bias).cuda()
        ids, w = torch.empty((3, k), dtype=torch.int32, device="cuda"), torch.empty((3, k), device="cuda")
        op = cb.ExpertRoute(E, k, score=kind)
        op.run(logits, ids, w, d_bias=b)
        check_route(torch, op, logits, b, ids, w, kind)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax", "sqrt_softplus"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,k,groups,top", [(384, 8, 8, 4), (96, 4, 32, 7), (352, 8, 11, 3)])
def test_route_groups_an_ulp_apart(cb, cuda, kind, with_bias, E, k, groups, top):
    torch = cuda
    per = E // groups
    for seed in range(6):
        rng = np.random.default_rng(seed * 77 + E)
        l = (rng.standard_normal((3, E)) * 2).astype(np.float32)
        bias = None
        first = np.concatenate([g * per + rng.permutation(per)[:2] for g in range(groups)])
        if with_bias:
            bias = close_bias(kind, l[0], first, rng)
        else:  # the same two logits on top of every group, an ulp apart here and there
            l[0] = np.minimum(l[0], 1.0)
            l[0][first] = np.tile(np.array([2.5, 2.0], np.float32), groups)
            l[0][first] += (rng.integers(-1, 2, 2 * groups) * np.spacing(np.float32(2.5))).astype(np.float32)
        logits = torch.from_numpy(l).cuda()
        b = None if bias is None else torch.from_numpy(bias).cuda()
        ids, w = torch.empty((3, k), dtype=torch.int32, device="cuda"), torch.empty((3, k), device="cuda")
        op = cb.ExpertRoute(E, k, score=kind, n_groups=groups, top_groups=top)
        op.run(logits, ids, w, d_bias=b)
        check_route(torch, op, logits, b, ids, w, kind, groups, top, True)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax", "sqrt_softplus"])
@pytest.mark.parametrize("pair", [True, False])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("E,k,groups", [(96, 16, 2), (64, 8, 32), (104, 15, 4), (384, 8, 8)])
def test_route_all_groups_stay(cb, cuda, kind, pair, with_bias, E, k, groups):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(E + k)
    logits = torch.randn((70, E), generator=gen, device="cuda") * 2
    logits[torch.rand((70, E), generator=gen, device="cuda") < 0.2] = -math.inf
    logits[3] = -math.inf
    logits[5, 9] = math.nan
    b = torch.randn(E, generator=gen, device="cuda") * 0.1 if with_bias else None
    ids, w = torch.empty((70, k), dtype=torch.int32, device="cuda"), torch.empty((70, k), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    op = cb.ExpertRoute(E, k, score=kind, n_groups=groups, top_groups=groups, group_score="pair" if pair else "max")
    op.run(logits, ids, w, d_bias=b, d_status=status)
    assert check_route(torch, op, logits, b, ids, w, kind, groups, groups, pair) == 1 and int(status) == 1


@pytest.mark.parametrize("kind", ["sigmoid", "softmax", "sqrt_softplus"])
@pytest.mark.parametrize("E,k", [(40, 4), (33, 16), (384, 8), (1024, 2)])
def test_route_close_picks_and_a_far_rest(cb, cuda, kind, E, k):
    """Two picks that fp32 cannot tell apart and everyone else far below: exactly k candidates."""
    torch = cuda
    rng = np.random.default_rng(E)
    l = np.full((2, E), -3.0, np.float32) + rng.standard_normal((2, E)).astype(np.float32) * 0.1
    first = rng.permutation(E)[:k]
    l[:, first] = 1.0 + 0.25 * np.arange(k, dtype=np.float32)
    bias = np.zeros(E, np.float32)
    held = scores64(kind, l[0].astype(np.float64)).astype(np.float32)
    bias[first[0]] = held[first[1]] - held[first[0]]
    logits, b = torch.from_numpy(l).cuda(), torch.from_numpy(bias).cuda()
    ids, w = torch.empty((2, k), dtype=torch.int32, device="cuda"), torch.empty((2, k), device="cuda")
    op = cb.ExpertRoute(E, k, score=kind)
    op.run(logits, ids, w, d_bias=b)
    check_route(torch, op, logits, b, ids, w, kind)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax", "sqrt_softplus"])
@pytest.mark.parametrize("mean", [-60.0, -14.0, -3.0, 9.0])
def test_route_small_and_close_scores(cb, cuda, kind, mean):
    """Scores all tiny or all close to 1, and biases of the size of their last bits."""
    torch = cuda
    E, k = 320, 8
    for seed in range(6):
        rng = np.random.default_rng(seed * 31 + 5)
        l = (rng.standard_normal((9, E)) * 0.01 + mean).astype(np.float32)
        held = scores64(kind, l[0].astype(np.float64)).astype(np.float32)
        bias = (rng.integers(-3, 4, E) * np.spacing(held.max())).astype(np.float32)
        bias[rng.random(E) < 0.3] *= np.float32(0.37)
        logits, b = torch.from_numpy(l).cuda(), torch.from_numpy(bias).cuda()
        for groups, top in ((1, 1), (8, 3)):
            ids, w = torch.empty((9, k), dtype=torch.int32, device="cuda"), torch.empty((9, k), device="cuda")
            op = cb.ExpertRoute(E, k, score=kind, n_groups=groups, top_groups=top)
            op.run(logits, ids, w, d_bias=b)
            check_route(torch, op, logits, b, ids, w, kind, groups, top, True)


@pytest.mark.parametrize("kind", ["sigmoid", "softmax", "sqrt_softplus"])
def test_route_huge_and_tiny_logits(cb, cuda, kind):
    torch = cuda
    E, k = 64, 8
    big = torch.finfo(torch.float32).max
    l = torch.zeros((6, E), device="cuda")
    l[0] = torch.linspace(-1, 1, E, device="cuda") * big   # differences that pass fp32
    l[1] = -big
    l[1, 7] = big
    l[2] = 1e-42
    l[2, 9] = -1e-42
    l[3] = torch.linspace(-300, 300, E, device="cuda")
    l[4] = -200.0
    l[4, ::2] = -201.0
    l[5] = big
    for bias in (None, torch.linspace(0.1, -0.1, E, device="cuda")):
        ids, w = torch.empty((6, k), dtype=torch.int32, device="cuda"), torch.empty((6, k), device="cuda")
        op = cb.ExpertRoute(E, k, score=kind, renormalize=False)
        op.run(l, ids, w, d_bias=bias)
        check_route(torch, op, l, bias, ids, w, kind, renorm=False)


def test_route_agrees_with_the_modes_there_were(cb, cuda):
    """Sigmoid without a bias is mode 0's choice; sqrt-softplus with a bias is mode 1's."""
    torch = cuda
    T, E, k = 513, 384, 6
    gen = torch.Generator(device="cuda").manual_seed(11)
    logits = torch.randn((T, E), generator=gen, device="cuda") * 2
    bias = torch.randn(E, generator=gen, device="cuda") * 0.1
    new = lambda d: torch.empty((T, k), dtype=d, device="cuda")  # noqa: E731
    a, aw, b, bw = new(torch.int32), new(torch.float32), new(torch.int32), new(torch.float32)
    cb.route_device(logits, E, k, T, a, aw)
    cb.ExpertRoute(E, k).run(logits, b, bw)
    assert torch.equal(a, b) and torch.allclose(aw, bw, rtol=(2 * k + 26) * U, atol=0)  # (k + 4) u and (2 * 9 + k + 4) u
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    cb.route_b_device(logits, bias, k, 2.5, a, aw, st)
    cb.ExpertRoute(E, k, score="sqrt_softplus", scale=2.5).run(logits, b, bw, d_bias=bias)
    # mode 1 rounds exp and log1p one after the other: its scores may be an ulp or two (4 u) apart
    same = (a == b).all(dim=1)
    assert float(same.float().mean()) > 0.999
    assert torch.allclose(aw[same], bw[same], rtol=(2 * k + 34) * U, atol=0)


# ------------------------------------------------------------------------------ norms

def norm64(h, y, g, w_post, w_pre, post, gate, sig, r, b, eps):
    """(h', x, r h, b g z) in 64 bits."""
    D = h.shape[1]
    rh, bz = h, np.zeros_like(h)
    if y is not None:
        z = y
        if post:
            z = y / np.sqrt((y * y).sum(1, keepdims=True) / D + eps) * (1.0 if w_post is None else w_post)
        if g is not None:
            g = 1.0 / (1.0 + np.exp(-g)) if sig else g
            z = z * (g[:, None] if gate == "token" else g)
        rh, bz = r * h, b * z
    new = rh + bz
    x = new / np.sqrt((new * new).sum(1, keepdims=True) / D + eps) * (1.0 if w_pre is None else w_pre)
    return new, x, rh, bz


def check_norm(torch, got, want, parts, D, dtype, inv_w=None):
    """Roundings: a row's sum of squares is a chain of at most 128 products and additions per
    thread (dim <= 32768) and 10 tree additions; its root's reciprocal halves that relative
    error and adds 6 operations of its own: (138 / 2 + 6) u = 75 u. z takes it once and 5 more
    products, a sigmoid gate 8 u (expf within 2 ulp, an addition, a division), h' two
    roundings. x takes the error of h' and its own root."""
    rh, bz = parts
    err_h = 90 * U * (np.abs(rh) + np.abs(bz))
    u_t = half_step(torch, dtype)
    if inv_w is None:
        tol = err_h + (u_t + U) * np.abs(want)
    else:
        # a relative change of every h' by at most e changes the root by e * |h'|'s own share
        share = np.sqrt((err_h ** 2).sum(1, keepdims=True) / np.maximum((inv_w[1] ** 2).sum(1, keepdims=True), 1e-300))
        tol = err_h * np.abs(inv_w[0]) + (share + 80 * U + u_t) * np.abs(want)
    tol = 1.01 * tol + TINY[dtype]
    assert np.all(np.isfinite(want))
    assert np.all(np.abs(got - want) <= tol), (np.abs(got - want) / tol).max()


def run_norm(cb, torch, T, D, h_t="float32", y_t="float32", x_t="float32", gate="none", sig=False, post=True, pre=True,
             weights=True, pad=0, seed=1, with_y=True, in_place=False, r=0.75, b=1.25, eps=1e-5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    dt = lambda n: getattr(torch, n)  # noqa: E731
    h = pitched(torch, rnd(T, D) * 3, dt(h_t), pad)
    y = pitched(torch, rnd(T, D) * 0.4, dt(y_t), pad) if with_y else None
    shape = {"none": None, "channel": (D,), "token": (T,), "full": (T, D)}[gate]
    g = None if shape is None or not with_y else rnd(*shape).to(dt(y_t))
    if gate == "full" and g is not None:
        g = pitched(torch, g, dt(y_t), pad)
    w_post = 1 + 0.3 * rnd(D) if post and weights and with_y else None
    w_pre = 1 + 0.3 * rnd(D) if pre and weights else None
    h64 = h.double().cpu().numpy()
    h_out = None if not with_y else h if in_place else pitched(torch, rnd(T, D), dt(h_t), pad)
    x = pitched(torch, rnd(T, D), dt(x_t), pad) if pre else None
    op = cb.BlockNorm(D, post=post, pre=pre, eps=eps, gate=gate if with_y else "none", gate_sigmoid=sig,
                      residual_scale=r, block_scale=b)
    op.run(h, d_y=y, d_gate=g, d_w_post=w_post, d_w_pre=w_pre, d_h_out=h_out, d_x=x)
    n64 = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    new, xw, rh, bz = norm64(h64, n64(y), n64(g), n64(w_post), n64(w_pre), post, gate, sig, r, b, eps)
    if with_y:
        check_norm(torch, n64(h_out), new, (rh, bz), D, h_t)
    if pre:
        inv = np.abs(xw) / np.maximum(np.abs(new), 1e-300)
        check_norm(torch, n64(x), xw, (rh, bz), D, x_t, (inv, new))
    for t in (h_out, x):  # what lies between the rows stays
        if t is not None and pad:
            assert bool((t._base[:, D:] == 7).all())
    return h_out, x


@pytest.mark.parametrize("D", [1, 7, 8, 64, 100, 1000, 2047, 2311, 5120, 7168, 8192, 8200, 16384, 16391, 32768])
@pytest.mark.parametrize("T", [1, 3, 150])
def test_norm_widths(cb, cuda, T, D):
    run_norm(cb, cuda, T, D, gate="channel")


@pytest.mark.parametrize("h_t", TYPES)
@pytest.mark.parametrize("y_t", TYPES)
@pytest.mark.parametrize("x_t", TYPES)
def test_norm_types(cb, cuda, h_t, y_t, x_t):
    run_norm(cb, cuda, 5, 768, h_t, y_t, x_t, gate="full", sig=True, seed=2)
    run_norm(cb, cuda, 300, 331, h_t, y_t, x_t, gate="full", sig=True, seed=3)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("sig", [False, True])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("D", [512, 515])
def test_norm_parts(cb, cuda, gate, sig, post, pre, D):
    run_norm(cb, cuda, 37, D, gate=gate, sig=sig, post=post, pre=pre, y_t="bfloat16")


@pytest.mark.parametrize("pad", [1, 4, 5, 8])
@pytest.mark.parametrize("h_t", ["float32", "bfloat16"])
def test_norm_pitches(cb, cuda, pad, h_t):
    run_norm(cb, cuda, 33, 1024, h_t, "float16", "bfloat16", gate="full", pad=pad)


@pytest.mark.parametrize("T,D", [(3, 1024), (400, 1024), (400, 1025)])
@pytest.mark.parametrize("h_t,y_t", [("float32", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16")])
def test_norm_rows_that_start_anywhere(cb, cuda, T, D, h_t, y_t):
    """Tensors whose first element is one past an aligned address."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(6)
    dt = lambda n: getattr(torch, n)  # noqa: E731
    at = lambda t, n: torch.randn((T, D + 9), generator=gen, device="cuda").to(dt(t))[:, n:n + D]  # noqa: E731
    h, y, g, out, x = at(h_t, 1), at(y_t, 3), at(y_t, 0), at(h_t, 8), at(y_t, 5)
    wide = torch.randn(D + 1, generator=gen, device="cuda")
    w_post, w_pre = wide[1:], wide[:D]
    cb.BlockNorm(D, eps=1e-5, gate="full").run(h, d_y=y, d_gate=g, d_w_post=w_post, d_w_pre=w_pre, d_h_out=out, d_x=x)
    n64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    new, xw, rh, bz = norm64(n64(h), n64(y), n64(g), n64(w_post), n64(w_pre), True, "full", False, 1.0, 1.0, 1e-5)
    check_norm(torch, n64(out), new, (rh, bz), D, h_t)
    check_norm(torch, n64(x), xw, (rh, bz), D, y_t, (np.abs(xw) / np.maximum(np.abs(new), 1e-300), new))


@pytest.mark.parametrize("D", [1, 2, 3, 4, 5, 7, 12, 30, 127, 1001, 1002, 1003, 2311, 8190, 8191, 9001, 16387, 20002, 32765])
@pytest.mark.parametrize("h_t,y_t,x_t", [("float32", "float32", "float32"), ("bfloat16", "bfloat16", "bfloat16"),
                                         ("float32", "float16", "float16"), ("float16", "float32", "bfloat16")])
def test_norm_rows_of_whole_fours(cb, cuda, D, h_t, y_t, x_t):
    """Rows that start at a multiple of four elements but not of eight; widths with 0 to 3 behind the last four."""
    norm_of_parts(cb, cuda, D, h_t, y_t, x_t, -D % 8 + 4)


@pytest.mark.parametrize("D", [1, 2, 3, 4, 6, 9, 30, 127, 822, 1001, 2310, 2311, 8190, 8191, 9002, 16387, 32766])
@pytest.mark.parametrize("h_t,y_t,x_t", [("float32", "float32", "float32"), ("bfloat16", "bfloat16", "bfloat16"),
                                         ("float32", "float16", "float16"), ("float16", "float32", "bfloat16")])
def test_norm_rows_of_whole_pairs(cb, cuda, D, h_t, y_t, x_t):
    norm_of_parts(cb, cuda, D, h_t, y_t, x_t, -D % 4 + 2)


def norm_of_parts(cb, cuda, D, h_t, y_t, x_t, pad):
    run_norm(cb, cuda, 3, D, h_t, y_t, x_t, gate="full", sig=True, pad=pad, seed=4)
    run_norm(cb, cuda, 2, D, h_t, y_t, x_t, gate="channel", pad=pad, seed=5, in_place=True)
    run_norm(cb, cuda, 2, D, h_t, y_t, x_t, pad=pad, post=False, weights=False, seed=6)
    run_norm(cb, cuda, 2, D, h_t, y_t, x_t, pad=pad, pre=False, gate="token", seed=7)
    run_norm(cb, cuda, 2, D, h_t, y_t, x_t, pad=pad, post=False, with_y=False, seed=8)
    if D <= 2311:
        run_norm(cb, cuda, 700, D, h_t, y_t, x_t, gate="full", pad=pad, seed=9)


@pytest.mark.parametrize("T,D", [(3, 1024), (400, 1026), (5, 4)])
@pytest.mark.parametrize("h_t,y_t", [("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float32")])
def test_norm_rows_that_start_at_fours(cb, cuda, T, D, h_t, y_t):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(16)
    dt = lambda n: getattr(torch, n)  # noqa: E731
    pitch = (D + 3) // 4 * 4 + 12
    at = lambda t, n: torch.randn((T, pitch), generator=gen, device="cuda").to(dt(t))[:, n:n + D]  # noqa: E731
    h, y, g, out, x = at(h_t, 4), at(y_t, 12), at(y_t, 0), at(h_t, 8), at(y_t, 4)
    before = x._base.clone()
    wide = torch.randn(D + 4, generator=gen, device="cuda")
    w_post, w_pre = wide[4:], wide[:D]
    cb.BlockNorm(D, eps=1e-5, gate="full").run(h, d_y=y, d_gate=g, d_w_post=w_post, d_w_pre=w_pre, d_h_out=out, d_x=x)
    n64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    new, xw, rh, bz = norm64(n64(h), n64(y), n64(g), n64(w_post), n64(w_pre), True, "full", False, 1.0, 1.0, 1e-5)
    check_norm(torch, n64(out), new, (rh, bz), D, h_t)
    check_norm(torch, n64(x), xw, (rh, bz), D, y_t, (np.abs(xw) / np.maximum(np.abs(new), 1e-300), new))
    keep = torch.ones(pitch, dtype=torch.bool, device="cuda")
    keep[4:4 + D] = False
    assert torch.equal(x._base[:, keep], before[:, keep])


@pytest.mark.parametrize("T", [999, 1000, 1001, 1007, 5000])
@pytest.mark.parametrize("D,pad", [(1, 0), (3, 1), (8, 0), (60, 4), (64, 2), (201, 0), (256, 0), (256, 1), (255, 5), (257, 0)])
def test_norm_many_short_rows(cb, cuda, T, D, pad):
    run_norm(cb, cuda, T, D, "float32", "bfloat16", "float16", gate="full", sig=True, pad=pad, seed=21)
    run_norm(cb, cuda, T, D, "bfloat16", "bfloat16", "bfloat16", gate="token", pad=pad, seed=22, in_place=True)
    run_norm(cb, cuda, T, D, "float16", "float16", "float16", gate="channel", pad=pad, seed=23, post=False)


@pytest.mark.parametrize("T", [1, 7, 500])
@pytest.mark.parametrize("D", [64, 100, 1024])
def test_norm_parts_of_one_buffer(cb, cuda, T, D):
    """h, y, h_out and x as columns of one buffer, whose rows interleave."""
    torch = cuda
    buf = torch.randn((T, 4 * D), generator=torch.Generator(device="cuda").manual_seed(T + D), device="cuda")
    h, y, out, x = (buf[:, i * D:(i + 1) * D] for i in range(4))
    keep = buf.clone()
    apart = [torch.empty((T, D), device="cuda") for _ in range(2)]
    op = cb.BlockNorm(D)
    op.run(h.contiguous(), d_y=y.contiguous(), d_h_out=apart[0], d_x=apart[1])
    op.run(h, d_y=y, d_h_out=out, d_x=x)
    for got, want in ((out, apart[0]), (x, apart[1])):  # the scalar and the aligned kernel add in another order
        assert torch.allclose(got, want, rtol=2.0 ** -18, atol=1e-6)
    assert torch.equal(buf[:, :2 * D], keep[:, :2 * D])
    if T > 1:
        with pytest.raises(cb.ClbError):
            op.run(h, d_y=y, d_h_out=buf[:, D // 2:D // 2 + D], d_x=x)


def test_no_tokens(cb, cuda):
    torch = cuda
    z = lambda n, t=torch.float32: torch.empty((0, n), dtype=t, device="cuda")  # noqa: E731
    cb.BlockNorm(64).run(z(64), d_y=z(64), d_h_out=z(64), d_x=z(64))
    w = torch.zeros((8, 64), dtype=torch.int8, device="cuda")
    lin = cb.Int8Linear(w, torch.zeros(8, device="cuda"))
    lin.run(z(64), z(8), d_ws=torch.empty(lin.workspace_bytes(0), dtype=torch.uint8, device="cuda"))
    lin.run(z(64, torch.int8), z(8), d_x_scale=torch.empty(0, device="cuda"))
    cb.int8_quantize(z(64), z(64, torch.int8), torch.empty(0, device="cuda"))


def test_norm_past_32_bits(cb, cuda):
    """Rows whose offsets in elements and bytes pass 2^32 (bf16, 131073 rows, 32768 apart)."""
    torch = cuda
    T, D, pitch = 131073, 64, 32768
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of free memory")
    h = torch.empty((T, pitch), dtype=torch.bfloat16, device="cuda")
    x = torch.empty((T, pitch), dtype=torch.bfloat16, device="cuda")
    h[:, :D] = torch.randn((T, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    cb.BlockNorm(D, post=False).run(h[:, :D], d_x=x[:, :D])
    few = torch.empty((64, D), dtype=torch.bfloat16, device="cuda")
    cb.BlockNorm(D, post=False).run(h[-64:, :D].contiguous(), d_x=few)
    # another kernel for few rows: each within one rounding of the exact value
    assert torch.allclose(x[-64:, :D].float(), few.float(), rtol=2.0 ** -7, atol=0)
    logits = h[:, :D]
    ids, w = torch.empty((T, 4), dtype=torch.int32, device="cuda"), torch.empty((T, 4), device="cuda")
    cb.ExpertRoute(D, 4).run(logits, ids, w)
    assert torch.equal(ids[-64:].long(), torch.sort(logits[-64:].float(), dim=1, descending=True, stable=True).indices[:, :4])


# calls of more than 1.6 million values, aligned rows: the kernel whose CTAs stay
LONG = [(210000, 8), (26000, 64), (13001, 128), (6600, 256), (6601, 264), (3301, 512), (3200, 520), (1701, 1024), (850, 2048),
        (790, 2056), (420, 4096), (331, 5120), (301, 5640), (235, 7168), (225, 7176), (203, 8192), (199, 8200), (101, 16384)]


@pytest.mark.parametrize("T,D", LONG)
def test_norm_many_rows(cb, cuda, T, D):
    run_norm(cb, cuda, T, D, gate="channel", sig=True, seed=8)
    run_norm(cb, cuda, T, D, "bfloat16", "bfloat16", "bfloat16", gate="full", seed=9)


@pytest.mark.parametrize("h_t,y_t,x_t", [("float32", "float32", "float32"), ("bfloat16", "bfloat16", "bfloat16"),
                                         ("float16", "float16", "float16"), ("float32", "bfloat16", "bfloat16"),
                                         ("float32", "float16", "float16"), ("bfloat16", "float16", "float32"),
                                         ("float16", "float32", "bfloat16"), ("bfloat16", "float32", "float32")])
@pytest.mark.parametrize("T,D", [(3300, 512), (420, 4096), (330, 5120), (235, 7168), (205, 8192)])
def test_norm_many_rows_types(cb, cuda, T, D, h_t, y_t, x_t):
    run_norm(cb, cuda, T, D, h_t, y_t, x_t, gate="full", sig=True, seed=10)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post,pre", [(True, True), (True, False), (False, True), (False, False)])
def test_norm_many_rows_parts(cb, cuda, gate, post, pre):
    run_norm(cb, cuda, 1700, 1024, y_t="bfloat16", gate=gate, sig=gate != "channel", post=post, pre=pre, pad=8, seed=11)
    run_norm(cb, cuda, 240, 7168, gate=gate, sig=True, post=post, pre=pre, seed=12)


def test_norm_many_rows_alone_and_in_place(cb, cuda):
    torch = cuda
    run_norm(cb, cuda, 3400, 512, with_y=False, x_t="bfloat16", seed=13)
    run_norm(cb, cuda, 3400, 512, weights=False, seed=14)
    a = run_norm(cb, cuda, 260, 7168, in_place=True, seed=15)
    b = run_norm(cb, cuda, 260, 7168, in_place=False, seed=15)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    T, D = 2000, 1024
    h = torch.randn((T, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    y = torch.randn((T, D), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    outs = [torch.empty((T, D), device="cuda") for _ in range(4)]
    op = cb.BlockNorm(D)
    op.run(h, d_y=y, d_h_out=outs[0], d_x=outs[1])
    y[7, 3], h[1999, 5], y[1000] = math.nan, math.inf, 0.0
    op.run(h, d_y=y, d_h_out=outs[2], d_x=outs[3])
    good = torch.ones(T, dtype=torch.bool, device="cuda")
    good[[7, 1000, 1999]] = False
    assert torch.equal(outs[0][good], outs[2][good]) and torch.equal(outs[1][good], outs[3][good])
    assert bool(torch.isnan(outs[3][7]).all()) and torch.equal(outs[2][1000], h[1000])
    assert bool(torch.isnan(outs[3][1999, 5])) and float(outs[2][1999, 5]) == math.inf


@pytest.mark.parametrize("gate_scale", [1.0, 20.0, 90.0])
@pytest.mark.parametrize("T", [40, 2000])
def test_norm_far_gates(cb, cuda, T, gate_scale):
    """Sigmoids of far arguments, in 16 bits (the fast form) and fp32. The fast form is off by at most
    (|g| + 8) u: 2^-17 for |g| <= 120, against half a step of 2^-9 (bf16) for the results; below
    -87.3 both forms may give 0 for a sigmoid under 2^-126, which is off by 2^-126 |y| after the
    product."""
    torch = cuda
    D = 1024
    gen = torch.Generator(device="cuda").manual_seed(T)
    for t in ("bfloat16", "float32"):
        dt = getattr(torch, t)
        h = torch.zeros((T, D), dtype=dt, device="cuda")
        y = torch.randn((T, D), generator=gen, device="cuda").to(dt)
        g = (torch.randn((T, D), generator=gen, device="cuda") * gate_scale).clamp_(-120, 120).to(dt)
        out = torch.empty_like(h)
        cb.BlockNorm(D, post=False, pre=False, gate="full", gate_sigmoid=True).run(h, d_y=y, d_gate=g, d_h_out=out)
        want = y.double() / (1 + torch.exp(-g.double()))
        tol = want.abs() * ((2.0 ** -17 + 2.0 ** -8) if t == "bfloat16" else 16 * U) + 2.0 ** -126 * y.double().abs() + TINY[t]
        assert bool(((out.double() - want).abs() <= tol).all())


def test_norm_without_weights_or_block(cb, cuda):
    run_norm(cb, cuda, 9, 1024, weights=False)
    run_norm(cb, cuda, 9, 7168, with_y=False)
    run_norm(cb, cuda, 2000, 640, with_y=False, x_t="bfloat16")


@pytest.mark.parametrize("T,D", [(1, 7168), (600, 1000), (5, 16384)])
def test_norm_in_place(cb, cuda, T, D):
    a = run_norm(cb, cuda, T, D, in_place=True, seed=4)
    b = run_norm(cb, cuda, T, D, in_place=False, seed=4)
    assert cuda.equal(a[0], b[0]) and cuda.equal(a[1], b[1])


def test_norm_zero_and_nonfinite_rows_stay_alone(cb, cuda):
    torch = cuda
    T, D = 6, 512
    gen = torch.Generator(device="cuda").manual_seed(5)
    h = torch.randn((T, D), generator=gen, device="cuda")
    y = torch.randn((T, D), generator=gen, device="cuda")
    clean_h, clean_x = torch.empty_like(h), torch.empty_like(h)
    op = cb.BlockNorm(D)
    op.run(h, d_y=y, d_h_out=clean_h, d_x=clean_x)
    h2, y2 = h.clone(), y.clone()
    y2[1] = 0.0
    h2[2], y2[2] = 0.0, 0.0
    y2[3, 5] = math.nan
    h2[4, 6] = math.inf
    out_h, out_x = torch.empty_like(h), torch.empty_like(h)
    op.run(h2, d_y=y2, d_h_out=out_h, d_x=out_x)
    assert torch.equal(out_h[[0, 5]], clean_h[[0, 5]]) and torch.equal(out_x[[0, 5]], clean_x[[0, 5]])
    assert torch.equal(out_h[1], h2[1])            # a zero row adds nothing: 0 / sqrt(eps)
    assert bool((out_h[2] == 0).all()) and bool((out_x[2] == 0).all())
    assert bool(torch.isnan(out_h[3]).all()) and bool(torch.isnan(out_x[3]).all())
    assert float(out_h[4, 6]) == math.inf and bool(torch.isnan(out_x[4, 6]))


# ------------------------------------------------------------------------------- int8

def quant64(x):
    """(q, scale) of rows by the definition: the scale held in fp32, the exact quotient's nearest integer."""
    m = np.abs(x).max(axis=1)
    s = (m / 127.0).astype(np.float32)
    bad = ~np.isfinite(m)
    d = np.where((s > 0) & ~bad, s, 1.0).astype(np.float64)[:, None]
    q = np.clip(np.rint(np.where(bad[:, None], 0.0, x) / d), -127, 127)
    q[(s == 0) | bad] = 0
    return q, np.where(bad, np.nan, s.astype(np.float64))


def padded_int8(torch, rows, k, extra=0):
    return torch.full((rows, (k + 15) // 16 * 16 + extra), 99, dtype=torch.int8, device="cuda")[:, :k]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,pad,extra", [(1, 1, 0, 0), (1, 7168, 0, 0), (3, 15, 1, 16), (5, 16, 0, 0), (9, 100, 5, 0),
                                              (300, 1536, 0, 0), (64, 2311, 3, 32), (7, 131072, 0, 0), (2, 20000, 8, 0)])
def test_quantize_exact(cb, cuda, dtype, rows, k, pad, extra):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows + k)
    x = torch.randn((rows, k), generator=gen, device="cuda")
    if rows > 4:
        x[1] = 0.0
        x[2] *= 2.0 ** -14
        x[3] = torch.round(x[3] * 8) * 0.5  # many quotients on or near a border
        x[3, 0] = 127.0
    x = pitched(torch, x, getattr(torch, dtype), pad)
    q, s = padded_int8(torch, rows, k, extra), torch.full((rows + 1,), -7.0, device="cuda")
    cb.int8_quantize(x, q, s[:rows])
    wq, ws = quant64(x.double().cpu().numpy())
    assert np.array_equal(s[:rows].double().cpu().numpy(), ws) and float(s[rows]) == -7
    assert np.array_equal(q.cpu().numpy(), wq.astype(np.int8))
    assert bool((q._base[:, k:] == 99).all())  # columns behind the row stay


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(3, 1), (3, 2), (3, 5), (3, 8), (3, 9), (3, 23), (3, 24), (5, 255), (5, 1001), (300, 1100),
                                    (2, 8195), (2, 12000), (2, 12019), (2, 12020), (2, 12050), (2, 24039), (2, 24041)])
def test_quantize_rows_that_start_anywhere(cb, cuda, dtype, rows, k):
    """Every first element within 32 bytes, and pitches that move the start from row to row; a NaN on both
    sides of each row shows any value that does not belong to it."""
    torch = cuda
    t = getattr(torch, dtype)
    gen = torch.Generator(device="cuda").manual_seed(k)
    values = torch.randn((rows, k), generator=gen, device="cuda").to(t)
    wq, ws = quant64(values.double().cpu().numpy())
    for first in range(1, 10 if k > 100 else 18):
        pitch = k + 2 + first % 3
        back = torch.full((first + rows * pitch + 8,), math.nan, dtype=t, device="cuda")
        x = back[first:first + rows * pitch].view(rows, pitch)[:, :k]
        x.copy_(values)
        q, s = padded_int8(torch, rows, k), torch.empty(rows, device="cuda")
        cb.int8_quantize(x, q, s)
        assert np.array_equal(s.double().cpu().numpy(), ws), first
        assert np.array_equal(q.cpu().numpy(), wq.astype(np.int8)), first


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 100), (9, 256), (1499, 300), (1500, 300), (1501, 512), (1503, 513), (1500, 1000), (2000, 1024),
                                    (2001, 1025), (2000, 7), (1777, 1)])
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_quantize_many_short_rows(cb, cuda, dtype, rows, k, pad):
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(rows + k)
    x = torch.randn((rows, k), generator=gen, device="cuda")
    x[rows // 2] = 0.0
    x[rows // 3] *= 2.0 ** -120  # a subnormal scale; zeros in fp16
    x[rows - 1] = torch.round(x[rows - 1] * 8) * 0.5
    x[rows - 1, 0] = 127.0
    if rows > 4:
        x[1, k - 1] = math.inf
    x = pitched(torch, x, getattr(torch, dtype), pad)
    q, s = padded_int8(torch, rows, k, 16), torch.full((rows + 1,), -7.0, device="cuda")
    cb.int8_quantize(x, q, s[:rows])
    wq, ws = quant64(x.double().cpu().numpy())
    assert np.array_equal(s[:rows].double().cpu().numpy(), ws, equal_nan=True) and float(s[rows]) == -7
    assert np.array_equal(q.cpu().numpy(), wq.astype(np.int8))
    assert bool((q._base[:, k:] == 99).all())


def test_quantize_borders_and_small_scales(cb, cuda):
    """Quotients a rounding away from a half, exact halves, subnormal rows and scales."""
    torch = cuda
    rng = np.random.default_rng(2)
    rows, k = 400, 256
    x = np.zeros((rows, k), np.float32)
    for r in range(rows):
        m = np.float32(rng.uniform(1, 2) * 2.0 ** int(rng.integers(-148, 120)))
        s = np.float32(np.float64(m) / 127.0)
        half = (rng.integers(-127, 127, k) + 0.5) * np.float64(s)
        x[r] = half.astype(np.float32)  # the representable numbers next to the borders
        x[r, ::3] = np.nextafter(x[r, ::3], np.float32(np.inf))
        x[r, 1::3] = np.nextafter(x[r, 1::3], np.float32(-np.inf))
        x[r] = np.clip(x[r], -m, m)
        x[r, 7] = m
    q, s = padded_int8(torch, rows, k), torch.empty(rows, device="cuda")
    cb.int8_quantize(torch.from_numpy(x).cuda(), q, s)
    wq, ws = quant64(x.astype(np.float64))
    assert np.array_equal(s.double().cpu().numpy(), ws)
    assert np.array_equal(q.cpu().numpy(), wq.astype(np.int8))


def test_quantize_nonfinite_rows(cb, cuda):
    torch = cuda
    x = torch.randn((4, 64), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    x[1, 3], x[2, 60] = math.nan, -math.inf
    q, s = padded_int8(torch, 4, 64), torch.empty(4, device="cuda")
    cb.int8_quantize(x, q, s)
    wq, ws = quant64(x.double().cpu().numpy())
    assert np.array_equal(s.double().cpu().numpy(), ws, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), wq.astype(np.int8))


def linear_case(cb, torch, T, K, N, x_t="float32", out_t="float32", bias=False, pad=0, seed=0, ready=False, extra=0,
                bad_row=None):
    gen = torch.Generator(device="cuda").manual_seed(seed + T + K + N)
    w = padded_int8(torch, N, K, extra)
    w.copy_(torch.randint(-127, 128, (N, K), generator=gen, device="cuda").to(torch.int8))
    ws = torch.rand(N, generator=gen, device="cuda") * 0.01 + 1e-4
    b = torch.randn(N, generator=gen, device="cuda") if bias else None
    x = torch.randn((T, K), generator=gen, device="cuda")
    if bad_row is not None:
        x[bad_row, K // 2] = math.nan
    back = torch.full((T + 1, N + pad), 7.0, dtype=getattr(torch, out_t), device="cuda")
    out = back[:T, :N]
    op = cb.Int8Linear(w, ws, b)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    if ready:
        q, xs = padded_int8(torch, T, K, extra), torch.empty(T, device="cuda")
        cb.int8_quantize(x, q, xs)
        op.run(q, out, d_x_scale=xs, d_status=status)
    else:
        x = pitched(torch, x, getattr(torch, x_t), pad)
        wsp = torch.empty(op.workspace_bytes(T), dtype=torch.uint8, device="cuda")
        op.run(x, out, d_ws=wsp, d_status=status)
    assert int(status) == 0
    wq, wxs = quant64(x.double().cpu().numpy())
    acc = (torch.from_numpy(wq).cuda() @ w.double().t()).cpu().numpy()  # integers below 2^53: exact
    v = acc * wxs[:, None] * ws.double().cpu().numpy()[None, :]
    want = v if b is None else v + b.double().cpu().numpy()[None, :]
    got = out.double().cpu().numpy()
    good = np.isfinite(wxs)
    assert np.all(np.isnan(got[~good]))
    # the sum to fp32, two products, the bias, the output type
    tol = 1.01 * (3 * U * np.abs(v) + (U + half_step(torch, out_t)) * np.abs(want)) + TINY[out_t]
    assert np.all(np.abs(got - want)[good] <= tol[good]), (np.abs(got - want)[good] / tol[good]).max()
    assert bool((back[T:] == 7).all()) and bool((back[:, N:] == 7).all())  # nothing behind the rows or the last row
    return out.clone()


@pytest.mark.parametrize("T", [1, 2, 3, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 128, 129, 255, 257, 500])
def test_linear_token_counts(cb, cuda, T):
    linear_case(cb, cuda, T, 1024, 768)


@pytest.mark.parametrize("K", [1, 15, 16, 17, 31, 100, 127, 128, 129, 255, 1000, 2311, 7168, 20000, 131072])
@pytest.mark.parametrize("T", [1, 6, 40, 300])
def test_linear_depths(cb, cuda, T, K):
    linear_case(cb, cuda, T, K, 136, extra=16 if K % 3 == 0 else 0)


@pytest.mark.parametrize("N", [1, 2, 31, 127, 128, 129, 250, 1001, 2304])
@pytest.mark.parametrize("T", [1, 5, 48, 270])
def test_linear_widths(cb, cuda, T, N):
    linear_case(cb, cuda, T, 512, N, out_t="bfloat16", bias=True)


@pytest.mark.parametrize("x_t", TYPES)
@pytest.mark.parametrize("out_t", TYPES)
@pytest.mark.parametrize("T", [1, 4, 20, 200])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_linear_types_and_pitches(cb, cuda, x_t, out_t, T, pad):
    linear_case(cb, cuda, T, 640, 300, x_t, out_t, bias=pad == 3, pad=pad)


@pytest.mark.parametrize("T", [1, 3, 12, 70, 300])
@pytest.mark.parametrize("K,extra", [(512, 0), (1000, 32)])
def test_linear_int8_input(cb, cuda, T, K, extra):
    a = linear_case(cb, cuda, T, K, 320, ready=True, extra=extra)
    b = linear_case(cb, cuda, T, K, 320, ready=False, extra=extra)
    assert cuda.equal(a, b)


@pytest.mark.parametrize("T", [1, 2, 30, 300])
def test_linear_nan_row_stays_alone(cb, cuda, T):
    linear_case(cb, cuda, T, 256, 200, bad_row=T // 2)


@pytest.mark.parametrize("T", [1, 3, 20, 300])
def test_linear_outputs_that_start_anywhere(cb, cuda, T):
    """16-bit outputs at odd elements and odd pitches, floating x one past an aligned address."""
    torch = cuda
    K, N = 264, 130
    gen = torch.Generator(device="cuda").manual_seed(T)
    w = padded_int8(torch, N, K)
    w.copy_(torch.randint(-127, 128, (N, K), generator=gen, device="cuda").to(torch.int8))
    op = cb.Int8Linear(w, torch.rand(N, generator=gen, device="cuda"))
    x = torch.randn((T, K + 3), generator=gen, device="cuda").to(torch.float16)
    ws = torch.empty(op.workspace_bytes(T), dtype=torch.uint8, device="cuda")
    want = torch.empty((T, N), dtype=torch.bfloat16, device="cuda")
    op.run(x[:, 1:1 + K].contiguous(), want, d_ws=ws)
    for pad, off in ((1, 0), (1, 1), (6, 1), (6, 2), (2, 0)):
        back = torch.full((T + 1, N + pad), 7.0, dtype=torch.bfloat16, device="cuda")
        out = back[:T, off:off + N]
        op.run(x[:, 1:1 + K], out, d_ws=ws)
        assert torch.equal(out, want), (pad, off)
        mask = torch.ones_like(back, dtype=torch.bool)
        mask[:T, off:off + N] = False
        assert bool((back[mask] == 7).all()), (pad, off)


@pytest.mark.parametrize("T", [1, 4, 9, 200])
def test_linear_lowest_int8(cb, cuda, T):
    """-128 on both sides, at the deepest K for which the sums cannot overflow."""
    torch = cuda
    K, N = 131071, 24
    back = torch.full((N, 131072), -128, dtype=torch.int8, device="cuda")
    q = torch.full((T, 131072), -128, dtype=torch.int8, device="cuda")
    out = torch.empty((T, N), device="cuda")
    cb.Int8Linear(back[:, :K], torch.ones(N, device="cuda")).run(q[:, :K], out, d_x_scale=torch.ones(T, device="cuda"))
    assert bool((out == float(np.float32(128 * 128 * K))).all())


@pytest.mark.parametrize("T", [1, 3, 20, 300])
@pytest.mark.parametrize("ready", [False, True])
def test_linear_sees_what_was_written_just_before(cb, cuda, T, ready):
    """Weights and tokens made by the calls in front, without a pause: a kernel that starts under
    the end of another must not read early."""
    torch = cuda
    K, N = 2048, 1536
    gen = torch.Generator(device="cuda").manual_seed(T)
    w, ws = torch.empty((N, K), dtype=torch.int8, device="cuda"), torch.empty(N, device="cuda")
    x, h = torch.empty((T, K), device="cuda"), torch.empty((T, K), device="cuda")
    q, qs = torch.empty((T, K), dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    lin, norm = cb.Int8Linear(w, ws), cb.BlockNorm(K, post=False)
    wsp = torch.empty(lin.workspace_bytes(T), dtype=torch.uint8, device="cuda")
    floats = [torch.randn((N, K), generator=gen, device="cuda") for _ in range(8)]
    inputs = [torch.randn((T, K), generator=gen, device="cuda") for _ in range(8)]
    outs = [[torch.empty((T, N), device="cuda") for _ in range(8)] for _ in range(2)]
    for wait, into in ((True, outs[0]), (False, outs[1])):
        pause = torch.cuda.synchronize if wait else lambda: None
        for i in range(8):
            h.copy_(inputs[i])
            pause()
            norm.run(h, d_x=x)
            pause()
            cb.int8_quantize(floats[i], w, ws)
            pause()
            if ready:
                cb.int8_quantize(x, q, qs)
                pause()
                lin.run(q, into[i], d_x_scale=qs)
            else:
                lin.run(x, into[i], d_ws=wsp)
            pause()
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a, b)


FIRST_CALL = """
import sys, torch
sys.path.insert(0, sys.argv[1])
import crosslane_b200 as cb
T, K, N = int(sys.argv[2]), 1024, 512
x, w = torch.randn((T, K), device="cuda"), torch.randint(-127, 128, (N, K), device="cuda").to(torch.int8)
lin = cb.Int8Linear(w, torch.ones(N, device="cuda"))
h, y = torch.randn((T, K), device="cuda"), torch.randn((T, K), device="cuda")
out, h2, x2 = torch.empty((T, N), device="cuda"), torch.empty_like(h), torch.empty_like(h)
ids, wts = torch.empty((T, 4), dtype=torch.int32, device="cuda"), torch.empty((T, 4), device="cuda")
ws = torch.empty(lin.workspace_bytes(T), dtype=torch.uint8, device="cuda")
norm, route = cb.BlockNorm(K), cb.ExpertRoute(64, 4)
def step():
    norm.run(h, d_y=y, d_h_out=h2, d_x=x2)
    route.run(h2[:, :64], ids, wts)
    lin.run(x2, out, d_ws=ws)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    step()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (h2, x2, ids, wts, out)]
for t in (h2, x2, wts, out):
    t.zero_()
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (h2, x2, ids, wts, out)))
print("captured first")
"""


@pytest.mark.parametrize("T", [1, 40, 400])
def test_first_call_inside_a_capture(cuda, T):
    """A process whose first calls are captured into a graph: the one-time set-up needs no eager call."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL, root, str(T)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_linear_past_32_bits(cb, cuda):
    """Weights whose offsets pass 2^31 bytes, outputs whose offsets pass 2^31 elements."""
    torch = cuda
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    K, N = 16384, 135000
    w = torch.empty((N, K), dtype=torch.int8, device="cuda")
    w.random_(-127, 128, generator=torch.Generator(device="cuda").manual_seed(1))
    op = cb.Int8Linear(w, torch.full((N,), 0.5, device="cuda"))
    for T in (1, 5, 40):
        q = torch.randint(-127, 128, (T, K), device="cuda").to(torch.int8)
        out = torch.empty((T, N), device="cuda")
        op.run(q, out, d_x_scale=torch.ones(T, device="cuda"))
        want = (q.double() @ w[-200:].double().t() * 0.5).float()
        assert torch.equal(out[:, -200:], want), T  # exact: sums below 2^24 or rounded once
    T, n = 16200, 135000
    small = cb.Int8Linear(torch.ones((n, 16), dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda"))
    out = torch.empty((T, n), dtype=torch.bfloat16, device="cuda")
    q = torch.ones((T, 16), dtype=torch.int8, device="cuda")
    q[-1] = 2
    small.run(q, out, d_x_scale=torch.ones(T, device="cuda"))
    assert bool((out[-1] == 32).all()) and bool((out[-2] == 16).all()) and bool((out[:, -1][:-1] == 16).all())


def test_calls_on_two_streams_at_once(cb, cuda):
    """Calls that overlap, with a workspace each, give the bits of calls one after the other."""
    torch = cuda
    K, N = 4096, 1024
    gen = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randint(-127, 128, (N, K), generator=gen, device="cuda").to(torch.int8)
    op = cb.Int8Linear(w, torch.rand(N, generator=gen, device="cuda"))
    jobs = []
    for i, T in enumerate((3, 40, 40, 700, 700, 64)):
        x = torch.randn((T, K), generator=gen, device="cuda")
        jobs.append((x, torch.empty((T, N), device="cuda"), torch.empty((T, N), device="cuda"),
                     torch.empty(op.workspace_bytes(T), dtype=torch.uint8, device="cuda"), torch.cuda.Stream()))
    for x, alone, _, ws, _ in jobs:
        op.run(x, alone, d_ws=ws)
    torch.cuda.synchronize()
    for _ in range(20):
        for x, _, out, ws, stream in jobs:
            op.run(x, out, d_ws=ws, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for _, alone, out, _, _ in jobs:
        assert torch.equal(alone, out)


def test_linear_extreme_sums(cb, cuda):
    """The largest integer sums: 127 * 127 * 131072 is below 2^31."""
    torch = cuda
    K, N = 131072, 40
    for T in (1, 5, 40):
        w = torch.full((N, K), 127, dtype=torch.int8, device="cuda")
        w[1::2] = -127
        q = torch.full((T, K), 127, dtype=torch.int8, device="cuda")
        out = torch.empty((T, N), device="cuda")
        cb.Int8Linear(w, torch.ones(N, device="cuda")).run(q, out, d_x_scale=torch.ones(T, device="cuda"))
        want = float(np.float32(127 * 127 * K))
        assert bool((out[:, ::2] == want).all()) and bool((out[:, 1::2] == -want).all())


def test_linear_does_not_depend_on_the_batch(cb, cuda):
    """A token's row has the same bits alone and in any batch (exact sums)."""
    torch = cuda
    K, N = 2048, 512
    gen = torch.Generator(device="cuda").manual_seed(9)
    w = torch.randint(-127, 128, (N, K), generator=gen, device="cuda").to(torch.int8)
    op = cb.Int8Linear(w, torch.rand(N, generator=gen, device="cuda"))
    x = torch.randn((600, K), generator=gen, device="cuda")
    ws = torch.empty(op.workspace_bytes(600), dtype=torch.uint8, device="cuda")
    full = torch.empty((600, N), device="cuda")
    op.run(x, full, d_ws=ws)
    for T in (1, 2, 5, 13, 40, 64, 150, 300):
        part = torch.empty((T, N), device="cuda")
        op.run(x[:T], part, d_ws=ws)
        assert torch.equal(part, full[:T]), T


# ----------------------------------------------------------- streams, graphs, the run of them

def test_streams_and_graphs(cb, cuda):
    """Another stream's calls, and a captured step replayed on new inputs, give the eager bits."""
    torch = cuda
    T, D, E, k, N = 24, 1024, 96, 4, 640
    gen = torch.Generator(device="cuda").manual_seed(21)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    w = torch.randint(-127, 128, (N, D), generator=gen, device="cuda").to(torch.int8)
    lin = cb.Int8Linear(w, torch.rand(N, generator=gen, device="cuda") * 0.01)
    route, norm = cb.ExpertRoute(E, k, n_groups=8, top_groups=4), cb.BlockNorm(D)
    bias = rnd(E) * 0.1
    s = dict(h=rnd(T, D), y=rnd(T, D), l=rnd(T, E), h2=rnd(T, D), x=rnd(T, D), o=rnd(T, N), w=rnd(T, k),
             ids=torch.empty((T, k), dtype=torch.int32, device="cuda"),
             ws=torch.empty(lin.workspace_bytes(T), dtype=torch.uint8, device="cuda"))

    def step():
        norm.run(s["h"], d_y=s["y"], d_h_out=s["h2"], d_x=s["x"])
        route.run(s["l"], s["ids"], s["w"], d_bias=bias)
        lin.run(s["x"], s["o"], d_ws=s["ws"])

    def outputs():
        torch.cuda.synchronize()
        return [s[n].clone() for n in ("h2", "x", "ids", "w", "o")]

    step()
    first = outputs()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for n in ("h2", "x", "o", "w"):
        s[n].zero_()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    for a, b in zip(first, outputs()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        g2 = torch.Generator(device="cuda").manual_seed(seed)
        for n in ("h", "y", "l"):
            s[n].copy_(torch.randn(s[n].shape, generator=g2, device="cuda"))
        step()
        want = outputs()
        for n in ("h2", "x", "o", "w"):
            s[n].fill_(-1)
        graph.replay()
        for a, b in zip(want, outputs()):
            assert torch.equal(a, b)


def test_moe_layer_with_its_norms_and_shared_expert(cb, orc, cuda):
    """One layer as a stage runs it: norm, router, routing, routed experts, the 8-bit shared
    expert, and the gated residual step with the next norm, against 64-bit arithmetic
    and the oracle's experts."""
    from oracle_lib import rel_l2
    torch = cuda
    T, dim, ff, E, k, seed, policy = 21, 2048, 512, 32, 4, 6, 2
    gen = torch.Generator(device="cuda").manual_seed(33)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    bank = cb.ExpertBank(n_layers=1, n_experts=E, dim=dim, ff=ff, max_picks=k, device=0)
    try:
        bank.fill_synthetic(seed, policy)
        h, w_pre, w_post, w_next = rnd(T, dim) * 2, 1 + 0.1 * rnd(dim), 1 + 0.1 * rnd(dim), 1 + 0.1 * rnd(dim)
        gate_w, bias, gate = rnd(E, dim) * 0.03, rnd(E) * 0.1, rnd(T)
        mats = {}
        for name, (n, kk) in {"gate": (ff, dim), "up": (ff, dim), "down": (dim, ff)}.items():
            q, sc = padded_int8(torch, n, kk), torch.empty(n, device="cuda")
            cb.int8_quantize(rnd(n, kk) * 0.05, q, sc)
            mats[name] = cb.Int8Linear(q, sc)
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        x, logits, ids, w = new(T, dim), new(T, E), torch.empty((T, k), dtype=torch.int32, device="cuda"), new(T, k)
        ws8 = torch.empty(max(m.workspace_bytes(T) for m in mats.values()), dtype=torch.uint8, device="cuda")
        g, u, a, shared, moe, h2, x2 = new(T, ff), new(T, ff), new(T, ff), new(T, dim), new(T, dim), new(T, dim), new(T, dim)
        pws = torch.empty(bank.prefill_workspace_bytes(T, k), dtype=torch.uint8, device="cuda")
        s = torch.cuda.current_stream().cuda_stream
        cb.BlockNorm(dim, post=False).run(h, d_w_pre=w_pre, d_x=x)
        cb.router_device(x, gate_w, logits)
        cb.ExpertRoute(E, k, n_groups=4, top_groups=2, scale=2.5).run(logits, ids, w, d_bias=bias)
        mats["gate"].run(x, g, d_ws=ws8)
        mats["up"].run(x, u, d_ws=ws8)
        cb.q8k_activate(g, u, a)
        mats["down"].run(a, shared, d_ws=ws8)
        torch.cuda.synchronize()  # the bank runs on its own stream here
        bank.prefill_layer_device(0, ids, w, x, moe, pws, d_resid=shared, stream=s or None)
        bank.synchronize()
        cb.BlockNorm(dim, gate="token", gate_sigmoid=True, block_scale=0.5).run(
            h, d_y=moe, d_gate=gate, d_w_post=w_post, d_w_pre=w_next, d_h_out=h2, d_x=x2)
        torch.cuda.synchronize()

        n = lambda t: t.double().cpu().numpy()  # noqa: E731
        xw = norm64(n(h), None, None, None, n(w_pre), False, "none", False, 1, 1, 1e-6)[1]
        assert rel_l2(n(x), xw) <= 1e-6
        check_route(torch, cb.ExpertRoute(E, k), logits, bias, ids, w, "sigmoid", 4, 2, True, True, 2.5)

        def lin64(m, v):
            q, sc = quant64(v)
            return (q @ m.d_w.double().cpu().numpy().T) * sc[:, None] * n(m.d_w_scale)[None, :]

        gw, uw = lin64(mats["gate"], n(x)), lin64(mats["up"], n(x))
        assert rel_l2(n(g), gw) <= 1e-6 and rel_l2(n(u), uw) <= 1e-6
        sw = lin64(mats["down"], n(a))
        assert rel_l2(n(a), n(g) / (1 + np.exp(-n(g))) * n(u)) <= 1e-6 and rel_l2(n(shared), sw) <= 1e-6
        xs, iw, ww = x.cpu().numpy(), ids.cpu().numpy(), w.cpu().numpy()
        routed = np.stack([orc.layer_synth(policy, seed, 0, iw[t], ww[t], xs[t], dim, ff) for t in range(T)])
        assert rel_l2(n(moe), routed.astype(np.float64) + n(shared)) <= 1e-3
        hw, x2w, _, _ = norm64(n(h), n(moe), n(gate), n(w_post), n(w_next), True, "token", True, 1.0, 0.5, 1e-6)
        assert rel_l2(n(h2), hw) <= 1e-6 and rel_l2(n(x2), x2w) <= 1e-6
    finally:
        bank.close()
