"""What the operators around the routed experts promise, as far as it shows without a GPU."""
import ctypes as C
import os

import pytest

import crosslane_b200 as cb
from crosslane_b200._capi import (BlockNormConfigV1, CLB_E_INVALID, ErrorV1, Int8LinearConfigV1, RouteConfigV1, lib)

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crosslane_b200", "csrc")


@pytest.mark.parametrize("name", ["clb_route.cu", "clb_block_norm.cu", "clb_int8.cu", "clb_ops.cuh", "clb_tc.cuh"])
def test_kernels_set_up_early_read_coherently(name):
    """A kernel whose CTAs start under the end of the one in front must not read what that one writes through the
    read-only path, whose data has to stay constant for the kernel's life."""
    with open(os.path.join(CSRC, name)) as f:
        code = "".join(line.split("//")[0] for line in f)
    assert "__ldg" not in code and "ld.global.nc" not in code and "__restrict__" not in code


M = 1 << 20  # buffers a megabyte apart; every call here is refused, so no address is ever used


def over(word, fn, *args):
    err = ErrorV1()
    assert fn(*args, None, C.byref(err)) == CLB_E_INVALID, (err.code, err.message)
    assert b"overlaps " + word.encode() in err.message, err.message


@pytest.mark.parametrize("kw,word", [
    (dict(ids=M), "logits"), (dict(ids=M + 4 * 64 * 8 - 4), "logits"), (dict(ids=M - 4 * 6 * 8 + 4), "logits"),
    (dict(w=M + 128), "logits"), (dict(ids=2 * M + 252), "bias"), (dict(w=2 * M), "bias"), (dict(w=3 * M), "weights"),
    (dict(ids=M, ld=1024), "logits")])
def test_route_refuses_outputs_over_inputs(kw, word):
    a = dict(logits=M, bias=2 * M, ids=3 * M, w=4 * M, ld=64)
    a.update(kw)
    cfg = RouteConfigV1(n_experts=64, k=6, n_groups=1, top_groups=1, group_score=2, renormalize=1, scale=1.0)
    over(word, lib.clb_route_experts_device, C.byref(cfg), a["logits"], a["ld"], a["bias"], 8, a["ids"], a["w"], None)


@pytest.mark.parametrize("kw,word", [
    (dict(h_out=3 * M), "gate"), (dict(x=3 * M + 8), "gate"), (dict(h_out=4 * M), "w_post"), (dict(x=5 * M + 252), "w_pre"),
    (dict(x=M), "h"), (dict(h_out=2 * M), "y"), (dict(x=6 * M), "x"), (dict(h_out=M, ld_h_out=72), "h"),
    (dict(gate=6 * M + 64, kind=2), "gate")])
def test_norm_refuses_outputs_over_inputs(kw, word):
    a = dict(h=M, y=2 * M, gate=3 * M, w_post=4 * M, w_pre=5 * M, h_out=6 * M, x=7 * M, kind=1, ld_h_out=64)
    a.update(kw)
    cfg = BlockNormConfigV1(dim=64, post=1, gate=a["kind"], post_eps=1e-6, pre_eps=1e-6, residual_scale=1.0, block_scale=1.0,
                            ld_h=64, ld_y=64, ld_gate=64, ld_h_out=a["ld_h_out"], ld_x=64)
    over(word, lib.clb_block_norm_device, C.byref(cfg), 8, a["h"], a["y"], a["gate"], a["w_post"], a["w_pre"], a["h_out"],
         a["x"])


@pytest.mark.parametrize("kw,word", [
    (dict(q=M), "x"), (dict(q=M, ld_q=256), "x"), (dict(scale=M + 64), "x"), (dict(scale=2 * M + 60), "scale"),
    (dict(q=M + 112, ld_q=512, ld_x=128), "x"), (dict(q=M + 240, ld_q=256), "x")])
def test_quantize_refuses_outputs_over_inputs(kw, word):
    a = dict(x=M, ld_x=64, q=2 * M, ld_q=64, scale=3 * M)
    a.update(kw)
    over(word, lib.clb_int8_quantize_device, 0, a["x"], a["ld_x"], 8, 64, a["q"], a["ld_q"], a["scale"])


@pytest.mark.parametrize("kw,word", [
    (dict(out=M), "x"), (dict(out=2 * M + 64), "w"), (dict(out=3 * M), "w_scale"), (dict(out=4 * M + 4), "bias"),
    (dict(out=5 * M + 64), "the workspace"), (dict(ws=M), "x"), (dict(ws=2 * M), "w"), (dict(ws=4 * M), "bias"),
    (dict(x_scale=6 * M, x_type=3, ws=None), "x_scale"), (dict(out=2 * M, ld_w=1 << 62, ld_out=1 << 61), "w")])
@pytest.mark.parametrize("tokens", [1, 8])
def test_linear_refuses_outputs_over_inputs(kw, word, tokens):
    a = dict(x=M, w=2 * M, w_scale=3 * M, bias=4 * M, ws=5 * M, out=6 * M, x_scale=None, x_type=0, ld_w=64, ld_out=32)
    a.update(kw)
    cfg = Int8LinearConfigV1(n=32, k=64, x_type=a["x_type"], ld_w=a["ld_w"], ld_x=64, ld_out=a["ld_out"])
    over(word, lib.clb_int8_linear_device, C.byref(cfg), a["w"], a["w_scale"], a["bias"], tokens, a["x"], a["x_scale"],
         a["out"], a["ws"], 1 << 16, None)


def test_linear_checks_its_own_tensors_at_every_call():
    """Scales, bias and weights that were replaced or changed in place behind a linear's back."""
    torch = pytest.importorskip("torch")

    def linear():
        return cb.Int8Linear(torch.zeros((8, 64), dtype=torch.int8), torch.zeros(8), torch.zeros(8))

    x, out = torch.zeros(4, 64), torch.zeros(4, 8)
    ws = torch.zeros(linear().workspace_bytes(4), dtype=torch.uint8)

    def refused_with(lin, word):
        with pytest.raises(cb.ClbError, match=word):
            lin.run(x, out, d_ws=ws)

    refused_with(linear(), "not on a CUDA device")  # nothing else is wrong with it
    for name, bad, word in (("d_w", torch.zeros((4, 64), dtype=torch.int8), "w is"), ("d_w", torch.zeros(8, 64), "w: "),
                            ("d_w_scale", torch.zeros(4), "w_scale"), ("d_w_scale", None, "w_scale"),
                            ("d_w_scale", torch.zeros(8).half(), "w_scale"), ("d_bias", torch.zeros(7), "bias")):
        lin = linear()
        setattr(lin, name, bad)
        refused_with(lin, word)
    lin = linear()
    lin.d_w_scale.resize_(3)
    refused_with(lin, "w_scale")
    lin = linear()
    lin.d_w.resize_(2, 64)
    refused_with(lin, "w is")


def test_wrappers_refuse_negated_views():
    """A view whose values torch negates as it reads them: its memory holds the opposite numbers."""
    torch = pytest.importorskip("torch")
    neg = torch.complex(torch.zeros(4, 1), torch.ones(4, 1)).conj().imag
    assert neg.is_neg() and float(neg[0, 0]) == -1
    with pytest.raises(cb.ClbError, match="negated"):
        cb.BlockNorm(1, post=False).run(neg, d_x=torch.zeros(4, 1))
    with pytest.raises(cb.ClbError, match="negated"):
        cb.BlockNorm(1, gate="token").run(torch.zeros(4, 1), d_y=torch.zeros(4, 1), d_gate=torch.zeros(4),
                                          d_h_out=torch.zeros(4, 1), d_x=neg)
    with pytest.raises(cb.ClbError, match="not on a CUDA device"):
        cb.BlockNorm(1, post=False).run(neg.resolve_neg(), d_x=torch.zeros(4, 1))
