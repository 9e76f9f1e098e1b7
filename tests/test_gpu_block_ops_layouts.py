"""How the operators around the routed experts are used together: inputs and outputs as columns of one buffer, a
whole layer on one stream."""
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


@pytest.mark.parametrize("T", [1, 21, 300])
def test_layer_on_one_stream(cb, cuda, T):
    """A layer's calls on a stream of their own, the bank's among them, without a pause: the bits of the same
    calls with a pause behind each. The layer's output is the next one's input."""
    torch = cuda
    dim, ff, E, k, layers = 2048, 512, 32, 4, 3
    gen = torch.Generator(device="cuda").manual_seed(T)
    rnd = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    bank = cb.ExpertBank(n_layers=layers, n_experts=E, dim=dim, ff=ff, max_picks=k, device=0)
    try:
        bank.fill_synthetic(6, 2)
        h0, gate_w, bias, tok_gate = rnd(T, dim) * 2, rnd(E, dim) * 0.03, rnd(E) * 0.1, rnd(T)
        mats = {}
        for name, (n, kk) in {"gate": (ff, dim), "up": (ff, dim), "down": (dim, ff)}.items():
            q, sc = torch.empty((n, kk), dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
            cb.int8_quantize(rnd(n, kk) * 0.05, q, sc)
            mats[name] = cb.Int8Linear(q, sc)
        norm_in, norm_out = cb.BlockNorm(dim, post=False), cb.BlockNorm(dim, gate="token", gate_sigmoid=True, block_scale=0.5)
        route = cb.ExpertRoute(E, k, n_groups=4, top_groups=2, scale=2.5)
        new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        ws = torch.empty(max(m.workspace_bytes(T) for m in mats.values()), dtype=torch.uint8, device="cuda")
        pws = torch.empty(bank.prefill_workspace_bytes(T, k), dtype=torch.uint8, device="cuda")
        stream = torch.cuda.Stream()
        results = []
        for pause in (torch.cuda.synchronize, lambda: None):
            h, x, logits, ids, w = h0.clone(), new(T, dim), new(T, E), torch.empty((T, k), dtype=torch.int32, device="cuda"), new(T, k)
            g, u, a, shared, moe = new(T, ff), new(T, ff), new(T, ff), new(T, dim), new(T, dim)
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                norm_in.run(h, d_x=x)
                for layer in range(layers):
                    for call in (lambda: cb.router_device(x, gate_w, logits), lambda: route.run(logits, ids, w, d_bias=bias),
                                 lambda: mats["gate"].run(x, g, d_ws=ws), lambda: mats["up"].run(x, u, d_ws=ws),
                                 lambda: cb.q8k_activate(g, u, a), lambda: mats["down"].run(a, shared, d_ws=ws),
                                 lambda: bank.prefill_layer_device(layer, ids, w, x, moe, pws, d_resid=shared,
                                                                   stream=stream.cuda_stream),
                                 lambda: norm_out.run(h, d_y=moe, d_gate=tok_gate, d_h_out=h, d_x=x)):
                        call()
                        pause()
            torch.cuda.synchronize()
            results.append((h, x, ids, w, moe))
        bank.synchronize()
        for got, want in zip(results[1], results[0]):
            assert torch.equal(got, want)
    finally:
        bank.close()
