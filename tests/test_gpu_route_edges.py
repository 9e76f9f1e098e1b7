"""Routing where its fast ranks are hardest to trust, against the definition of test_gpu_block_ops."""
import numpy as np
import pytest

from test_gpu_block_ops import check_route

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
