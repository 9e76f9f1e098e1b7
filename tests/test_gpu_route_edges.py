"""Routing where its fast ranks are hardest to trust: rows of the types' lowest values, identical
experts on both sides of the last pick, group values that cancel, scores far below the smallest
exponential, and logits written by the call in front. Against the definition of test_gpu_block_ops.
"""
import numpy as np
import pytest

from test_gpu_block_ops import check_route, scores64

pytestmark = pytest.mark.gpu

KINDS = ["sigmoid", "softmax", "sqrt_softplus"]


@pytest.fixture(scope="module")
def cb(cuda):
    import crosslane_b200
    return crosslane_b200


def run_and_check(cb, torch, logits, bias, k, kind, groups=1, top=1, pair=True, renorm=True):
    T, E = logits.shape
    ids = torch.full((T, k), -7, dtype=torch.int32, device="cuda")
    w = torch.full((T, k), -7.0, device="cuda")
    op = cb.ExpertRoute(E, k, score=kind, n_groups=groups, top_groups=top, group_score="pair" if pair else "max",
                        renormalize=renorm)
    op.run(logits, ids, w, d_bias=bias)
    assert check_route(torch, op, logits, bias, ids, w, kind, groups, top, pair, renorm) == 0
    return ids, w


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("E,k,groups,top", [(3, 2, 1, 1), (20, 6, 1, 1), (64, 8, 1, 1), (64, 8, 8, 8), (384, 6, 1, 1),
                                            (384, 8, 8, 4), (1024, 16, 1, 1)])
def test_route_rows_of_the_lowest_value(cb, cuda, kind, dtype, E, k, groups, top):
    """Padding rows filled with the type's lowest value, whole or in part: every score is 0 (softmax: the same),
    and the biases alone decide. Every id is distinct and in range."""
    torch = cuda
    t = getattr(torch, dtype)
    low = torch.finfo(t).min
    gen = torch.Generator(device="cuda").manual_seed(E + k)
    logits = torch.full((7, E), low, device="cuda")
    logits[1, ::2] = -np.inf
    logits[2, 0] = low / 2
    logits[3] *= torch.rand(E, generator=gen, device="cuda") * 0.5 + 0.5
    logits[4, 1] = 0.0
    logits[5, : max(1, E - k)] = -np.inf  # k left
    logits[6] = torch.randn(E, generator=gen, device="cuda")
    logits = logits.to(t)
    biases = [torch.randn(E, generator=gen, device="cuda") * 0.1, torch.linspace(0.2, -0.2, E, device="cuda"),
              torch.zeros(E, device="cuda")]
    biases[0][E // 2] = -np.inf
    for bias in biases:
        for renorm in (True, False):
            ids, _ = run_and_check(cb, torch, logits, bias, k, kind, groups, top, renorm=renorm)
            assert int(ids.min()) >= 0 and int(ids.max()) < E


def test_route_identical_experts_at_the_last_place(cb, cuda):
    """One pick of [16.4, 16.7, 16.7]: all three scores are 1 - 2^-24 in fp32, so the first expert is it."""
    torch = cuda
    logits = torch.full((2, 9), -4.0, device="cuda")
    logits[0, :3] = torch.tensor([16.4, 16.7, 16.7])
    logits[1, 5:8] = torch.tensor([16.7, 16.7, 16.4])
    ids, _ = run_and_check(cb, torch, logits, torch.zeros(9, device="cuda"), 1, "sigmoid")
    assert ids.flatten().tolist() == [0, 5]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("E,k,copies", [(40, 1, 2), (40, 3, 2), (384, 6, 2), (384, 8, 3), (384, 6, 50), (1000, 16, 2)])
@pytest.mark.parametrize("third_first", [True, False])
def test_route_twins_at_the_cut(cb, cuda, kind, E, k, copies, third_first):
    """k - 1 sure picks, then experts of one logit and one bias around the last place, and another whose rank is
    within an ulp of theirs, at a lower or a higher id."""
    torch = cuda
    for seed in range(40):
        rng = np.random.default_rng(seed * 100 + E + k)
        l = (rng.standard_normal(E) - 2.0).astype(np.float32)
        at = np.sort(rng.permutation(E)[:k + copies])
        sure, twins = at[:k - 1], at[k - 1:]
        third = twins[0] if third_first else twins[-1]
        twins = twins[1:] if third_first else twins[:-1]
        l[sure] = 2.5
        l[twins] = np.float32(rng.uniform(0.3, 1.5))
        l[third] = np.float32(rng.uniform(0.3, 1.5))
        held = scores64(kind, l.astype(np.float64)).astype(np.float32)
        bias = np.full(E, -2.0, np.float32)
        bias[sure] = 1.0
        bias[twins] = np.float32(rng.uniform(0.0, 0.4))
        rank = held[twins[0]] + bias[twins[0]]
        bias[third] = rank - held[third] + np.float32(rng.integers(-1, 2)) * np.spacing(rank)
        run_and_check(cb, torch, torch.from_numpy(l[None]).cuda(), torch.from_numpy(bias).cuda(), k, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("groups", [1, 4])
def test_route_constant_rows(cb, cuda, kind, groups):
    """Every expert the same: ascending ids."""
    torch = cuda
    logits = torch.zeros((5, 256), device="cuda")
    logits[1], logits[2], logits[3, ::3], logits[4, 200:] = 3.7, -20.0, 1.0, -np.inf
    for b in (0.0, 0.3, -1e9):
        run_and_check(cb, torch, logits, torch.full((256,), b, device="cuda"), 8, kind, groups, max(1, groups // 2))


def at_borders(kind, base, step, firsts, low, rng):
    """Logits whose scores at `firsts` lie a few ulps around the middle between two ranks of fp32, where ranks are
    `step` apart (multiples of it from `base` on)."""
    E = low.size
    l = low.astype(np.float64)
    want = np.empty(len(firsts))
    for i in range(len(firsts)):
        border = (np.floor(base / step) + 0.5) * step
        want[i] = border + rng.integers(-5, 6) * np.spacing(np.float32(border)).astype(np.float64)
    if kind == "sigmoid":
        l[firsts] = np.log(want / (1 - want))
    elif kind == "sqrt_softplus":
        l[firsts] = np.log(np.expm1(want * want))
    else:  # the firsts' share of the sum is known: the others keep theirs
        rest = np.exp(l[np.setdiff1d(np.arange(E), firsts)]).sum()
        l[firsts] = np.log(want * rest / (1 - want.sum()))
    return l.astype(np.float32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B", [1.0, 64.0, 1000.0, 1e6])
@pytest.mark.parametrize("groups,per,top", [(8, 2, 3), (8, 12, 3), (6, 12, 2)])
def test_route_group_values_that_cancel(cb, cuda, kind, B, groups, per, top):
    """A group's two best ranks are near +B and -B, so its value is small while each rank's rounding is a step of B;
    the first scores lie where that rounding turns."""
    torch = cuda
    rng = np.random.default_rng(int(B) + groups + per)
    E, T = groups * per, 300
    firsts, seconds = np.arange(groups) * per, np.arange(groups) * per + per - 1
    bias = np.full(E, -3 * B, np.float32)
    bias[firsts], bias[seconds] = B, -B
    step = float(np.spacing(np.float32(B + 0.03)))
    rows = []
    for _ in range(T):
        low = np.full(E, 0.5, np.float32)
        # a score that the firsts can all have at once (softmax), more than half a step of the largest B
        rows.append(at_borders(kind, 0.07 if kind == "softmax" else 0.3, step, firsts, low, rng))
    run_and_check(cb, torch, torch.from_numpy(np.stack(rows)).cuda(), torch.from_numpy(bias).cuda(), min(4, top * per),
                  kind, groups, top, True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pair", [True, False])
@pytest.mark.parametrize("mask", [-1e9, float(np.finfo(np.float32).min)])
def test_route_biases_that_mask(cb, cuda, kind, pair, mask):
    """Finite biases that put experts out of the running, one of a group, most of a group, whole groups."""
    torch = cuda
    gen = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn((50, 96), generator=gen, device="cuda")
    bias = torch.randn(96, generator=gen, device="cuda") * 0.1
    bias[3] = mask
    bias[13:24] = mask
    bias[24:48] = mask
    with np.errstate(over="ignore"):  # the definition adds two lowest values
        run_and_check(cb, torch, logits, bias, 6, kind, 8, 3, pair)
        bias[:90] = mask
        run_and_check(cb, torch, logits, bias, 6, kind, 8, 3, pair)


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("with_bias", [True, False])
def test_route_square_root_scores_far_below(cb, cuda, renorm, with_bias):
    """sqrt(softplus(l)) is e^(l/2) for very negative logits: a normal number down to l = -174, long after e^l is
    not."""
    torch = cuda
    E, k = 64, 8
    logits = torch.stack([torch.linspace(hi, hi - 4.0, E, device="cuda")
                          for hi in (-10.0, -18.0, -50.0, -80.0, -86.0, -88.0, -95.0, -100.0, -104.0, -120.0, -165.0, -400.0)])
    bias = torch.linspace(-0.1, 0.1, E, device="cuda") if with_bias else None
    run_and_check(cb, torch, logits, bias, k, "sqrt_softplus", renorm=renorm)


@pytest.mark.parametrize("T", [1, 33, 3000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_route_sees_what_was_written_just_before(cb, cuda, T, dtype):
    """Logits made by the call in front, without a pause, over those of the call before."""
    torch = cuda
    E, k = 256, 8
    gen = torch.Generator(device="cuda").manual_seed(T)
    op, norm = cb.ExpertRoute(E, k, score="softmax"), cb.BlockNorm(E, post=False)
    inputs = [torch.randn((T, E), generator=gen, device="cuda") for _ in range(8)]
    logits = torch.zeros((T, E), dtype=getattr(torch, dtype), device="cuda")
    runs = []
    for wait in (True, False):
        out = [(torch.empty((T, k), dtype=torch.int32, device="cuda"), torch.empty((T, k), device="cuda")) for _ in inputs]
        for x, (ids, w) in zip(inputs, out):
            norm.run(x, d_x=logits)
            if wait:
                torch.cuda.synchronize()
            op.run(logits, ids, w)
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        runs.append(out)
    for (a, aw), (b, bw) in zip(*runs):
        assert torch.equal(a, b) and torch.equal(aw, bw)
