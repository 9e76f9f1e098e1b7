"""Layouts that the operators around the routed experts allow: inputs and outputs as columns of one buffer."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cb(cuda):
    import crosslane_b200
    return crosslane_b200


@pytest.mark.parametrize("T", [1, 3, 40, 300])
def test_linear_columns_of_one_buffer(cb, cuda, T):
    torch = cuda
    K, N = 320, 200
    gen = torch.Generator(device="cuda").manual_seed(T)
    w = torch.randint(-127, 128, (N, K), generator=gen, device="cuda").to(torch.int8)
    lin = cb.Int8Linear(w, torch.rand(N, generator=gen, device="cuda"))
    ws = torch.empty(lin.workspace_bytes(T), dtype=torch.uint8, device="cuda")
    buf = torch.randn((T, K + N + 8), generator=gen, device="cuda")
    keep, want = buf.clone(), torch.empty((T, N), device="cuda")
    lin.run(buf[:, :K].contiguous(), want, d_ws=ws)
    lin.run(buf[:, :K], buf[:, K + 8:], d_ws=ws)
    assert torch.equal(buf[:, K + 8:], want) and torch.equal(buf[:, :K + 8], keep[:, :K + 8])


@pytest.mark.parametrize("T,K", [(1, 64), (5, 64), (300, 1104), (2000, 256), (3, 40000)])
def test_quantize_into_the_gaps_of_its_rows(cb, cuda, T, K):
    """Rows of fp32 with room behind each for the same values in 8 bits."""
    torch = cuda
    buf = torch.empty((T, 5 * K), dtype=torch.int8, device="cuda")
    x, q = buf.view(torch.float32)[:, :K], buf[:, 4 * K:]
    x.copy_(torch.randn((T, K), generator=torch.Generator(device="cuda").manual_seed(K), device="cuda"))
    keep, s = x.clone(), torch.empty(T, device="cuda")
    want, ws = torch.empty((T, K), dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")
    cb.int8_quantize(keep, want, ws)
    cb.int8_quantize(x, q, s)
    assert torch.equal(q, want) and torch.equal(s, ws) and torch.equal(x, keep)


def test_outputs_over_inputs_are_refused(cb, cuda):
    torch = cuda
    x = torch.randn((8, 64), device="cuda")
    with pytest.raises(cb.ClbError, match="overlaps"):  # in place: a row's bytes are read after another's are written
        cb.int8_quantize(x, x.view(torch.int8).view(-1)[:512].view(8, 64), torch.empty(8, device="cuda"))
    lin = cb.Int8Linear(torch.zeros((64, 64), dtype=torch.int8, device="cuda"), torch.zeros(64, device="cuda"))
    ws = torch.empty(lin.workspace_bytes(8), dtype=torch.uint8, device="cuda")
    with pytest.raises(cb.ClbError, match="overlaps"):
        lin.run(x, x, d_ws=ws)
    keep = x.clone()
    with pytest.raises(cb.ClbError, match="overlaps"):
        cb.BlockNorm(64, post=False).run(x, d_x=x)
    assert torch.equal(x, keep)
