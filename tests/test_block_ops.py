"""Argument checks of the operators around the routed experts (no GPU: every refusal comes
before the first CUDA call) and the torch wrappers' own."""
import ctypes as C

import pytest

import crosslane_b200 as cb
from crosslane_b200._capi import (BlockNormConfigV1, CLB_E_INVALID, CLB_OK, ErrorV1, Int8LinearConfigV1, RouteConfigV1,
                                  lib)

A = 1 << 20  # an aligned address that is never read: every call here is refused before a launch


def refused(fn, *args):
    err = ErrorV1()
    rc = fn(*args, None, C.byref(err))
    assert rc == CLB_E_INVALID and err.code == CLB_E_INVALID and err.message, (rc, err.message)


def route(tokens=4, ld=None, logits=A, ids=A, w=A, bias=None, status=None, **kw):
    base = dict(n_experts=64, k=6, score=0, n_groups=1, top_groups=1, group_score=2, renormalize=1, scale=1.0,
                logits_type=0)
    base.update(kw)
    cfg = RouteConfigV1(**base)
    return (lib.clb_route_experts_device, C.byref(cfg), logits, ld if ld is not None else cfg.n_experts, bias, tokens,
            ids, w, status)


@pytest.mark.parametrize("kw", [
    dict(n_experts=0), dict(n_experts=1025), dict(k=0), dict(k=17), dict(n_experts=4, k=5), dict(score=3), dict(score=-1),
    dict(n_groups=0), dict(n_groups=33), dict(n_groups=3), dict(n_groups=64), dict(n_groups=4, top_groups=5),
    dict(top_groups=0), dict(n_groups=16, top_groups=1), dict(n_groups=2, group_score=0), dict(renormalize=2),
    dict(scale=float("nan")), dict(scale=-1.0), dict(scale=float("inf")), dict(logits_type=3), dict(tokens=-1),
    dict(ld=63), dict(logits=None), dict(ids=None), dict(w=None), dict(logits=A + 2), dict(bias=A + 1), dict(ids=A + 2),
    dict(logits=A + 1, logits_type=1), dict(status=A + 1)])
def test_route_refusals(kw):
    refused(*route(**kw))


def test_route_refuses_null_config_and_reserved():
    refused(lib.clb_route_experts_device, None, A, 64, None, 4, A, A, None)
    fn, cfg, *rest = route()
    cfg._obj.reserved[1] = 1
    refused(fn, cfg, *rest)


def norm(tokens=4, h=A, y=2 * A, gate=None, w_post=None, w_pre=None, h_out=3 * A, x=4 * A, **kw):
    base = dict(dim=64, post=1, gate=0, post_eps=1e-6, pre_eps=1e-6, residual_scale=1.0, block_scale=1.0, ld_h=64,
                ld_y=64, ld_gate=64, ld_h_out=64, ld_x=64)
    base.update(kw)
    return (lib.clb_block_norm_device, C.byref(BlockNormConfigV1(**base)), tokens, h, y, gate, w_post, w_pre, h_out, x)


@pytest.mark.parametrize("kw", [
    dict(dim=0), dict(dim=32769), dict(post=2), dict(gate=4), dict(gate=-1), dict(h_type=3), dict(y_type=9),
    dict(x_type=-1), dict(post_eps=0.0), dict(pre_eps=-1.0), dict(pre_eps=float("nan")),
    dict(residual_scale=float("inf")), dict(block_scale=float("nan")), dict(tokens=-1), dict(h=None),
    dict(y=None, h_out=None, x=None), dict(y=None), dict(h_out=None), dict(y=None, h_out=None, gate=A, gate_=1),
    dict(y=None, h_out=None, w_post=5 * A), dict(gate=1), dict(w_post=5 * A, post=0), dict(w_pre=5 * A, x=None),
    dict(ld_h=63), dict(ld_y=0), dict(ld_x=10), dict(ld_h_out=63), dict(h=A + 2), dict(y=2 * A + 1, y_type=1),
    dict(w_pre=5 * A + 2), dict(x=A), dict(x=3 * A), dict(h_out=A, ld_h_out=72), dict(h_out=2 * A), dict(h_out=A + 256),
    dict(x=2 * A + 4 * 32)])
def test_norm_refusals(kw):
    kw = {k: v for k, v in kw.items() if k != "gate_"}
    if kw.get("gate") in (4, -1, 1):  # the kind in the config, no pointer
        fn, cfg, *rest = norm(**{k: v for k, v in kw.items() if k != "gate"})
        cfg._obj.gate = kw["gate"]
        refused(fn, cfg, *rest)
    else:
        refused(*norm(**kw))


def test_norm_refuses_a_narrow_full_gate():
    fn, cfg, *rest = norm(gate=5 * A, ld_gate=63)
    cfg._obj.gate = 3
    refused(fn, cfg, *rest)


@pytest.mark.parametrize("kw", [
    dict(type=3), dict(type=7), dict(k=0), dict(k=131073), dict(rows=-1), dict(ld_x=63), dict(ld_q=48), dict(ld_q=72),
    dict(x=None), dict(q=None), dict(scale=None), dict(x=A + 2), dict(q=A + 8), dict(scale=A + 2)])
def test_quantize_refusals(kw):
    a = dict(type=0, x=A, ld_x=64, rows=4, k=64, q=2 * A, ld_q=64, scale=3 * A)
    a.update(kw)
    if a["k"] > 64:
        a["ld_x"] = a["ld_q"] = 131088
    refused(lib.clb_int8_quantize_device, a["type"], a["x"], a["ld_x"], a["rows"], a["k"], a["q"], a["ld_q"], a["scale"])


@pytest.mark.parametrize("kw", [
    dict(n=0), dict(k=0), dict(k=131073, ld_w=131088, ld_x=131088), dict(x_type=4), dict(out_type=3), dict(ld_w=48),
    dict(ld_w=72), dict(ld_x=63), dict(ld_out=31), dict(tokens=-1), dict(w=None), dict(w_scale=None), dict(x=None),
    dict(out=None), dict(w=A + 8), dict(x=A + 2), dict(out=A + 2), dict(ws=None), dict(ws=A + 8), dict(ws_bytes=4 * 64),
    dict(x_scale=A), dict(x_type=3), dict(x_type=3, x_scale=A, ld_x=72), dict(x_type=3, x_scale=A, x=A + 8),
    dict(bias=A + 1), dict(status=A + 1)])
def test_linear_refusals(kw):
    a = dict(w=A, w_scale=A, bias=None, tokens=4, x=A, x_scale=None, out=A, ws=A, ws_bytes=1 << 20, status=None)
    base = dict(n=32, k=64, x_type=0, out_type=0, ld_w=64, ld_x=64, ld_out=32)
    for k, v in kw.items():
        (base if k in base else a)[k] = v
    cfg = Int8LinearConfigV1(**base)
    refused(lib.clb_int8_linear_device, C.byref(cfg), a["w"], a["w_scale"], a["bias"], a["tokens"], a["x"],
            a["x_scale"], a["out"], a["ws"], a["ws_bytes"], a["status"])


@pytest.mark.parametrize("kw", [dict(n=(1 << 30) + 1, ld_out=(1 << 30) + 1), dict(n=2 ** 31 - 1, ld_out=2 ** 31 - 1),
                                dict(tokens=(1 << 30) + 1), dict(tokens=2 ** 31 - 1)])
def test_linear_refuses_more_rows_than_it_counts(kw):
    cfg = Int8LinearConfigV1(**{**dict(n=32, k=16, ld_w=16, ld_x=16, ld_out=32), **{k: v for k, v in kw.items() if k != "tokens"}})
    refused(lib.clb_int8_linear_device, C.byref(cfg), A, A, None, kw.get("tokens", 4), A, None, A, A, 1 << 62, None)


def test_zero_tokens_are_no_work():
    err = ErrorV1()
    for fn, *args in (route(tokens=0, logits=None, ids=None, w=None),
                      norm(tokens=0, h=None, y=None, h_out=None, x=None)):
        assert fn(*args, None, C.byref(err)) == CLB_OK and err.code == CLB_OK
    assert lib.clb_int8_quantize_device(0, None, 64, 0, 64, None, 64, None, None, None) == CLB_OK
    cfg = Int8LinearConfigV1(n=8, k=64, ld_w=64, ld_x=64, ld_out=8)
    assert lib.clb_int8_linear_device(C.byref(cfg), None, None, None, 0, None, None, None, None, 0, None, None,
                                      C.byref(err)) == CLB_OK


def test_workspace_bytes():
    assert lib.clb_int8_linear_workspace_bytes(-1, 64) == 0
    assert lib.clb_int8_linear_workspace_bytes(4, 0) == 0
    assert lib.clb_int8_linear_workspace_bytes(4, 131073) == 0
    for t, k in ((0, 64), (1, 1), (7, 33), (100000, 131072)):  # past 32 bits too
        assert lib.clb_int8_linear_workspace_bytes(t, k) >= t * ((k + 15) // 16 * 16) + 4 * t


def test_wrappers_refuse():
    torch = pytest.importorskip("torch")
    with pytest.raises(cb.ClbError):
        cb.ExpertRoute(64, 6, score="relu")
    with pytest.raises(cb.ClbError):
        cb.ExpertRoute(64, 6, n_groups=5)
    with pytest.raises(cb.ClbError):
        cb.BlockNorm(64, gate="row")
    with pytest.raises(cb.ClbError):
        cb.BlockNorm(0)
    r = cb.ExpertRoute(64, 6)
    t = torch.zeros(4, 64)
    ids, w = torch.zeros(4, 6, dtype=torch.int32), torch.zeros(4, 6)
    for bad in ((t.double(), ids, w), (t[:, :63], ids, w), (t, ids.long(), w), (t, ids[:3], w), (t, ids, w.half()),
                (t.t().contiguous().t(), ids, w), (t[0], ids, w), (t, ids, w)):  # the last: not on a GPU
        with pytest.raises(cb.ClbError):
            r.run(*bad)
    n = cb.BlockNorm(64)
    h, x = torch.zeros(4, 64), torch.zeros(4, 64)
    for kw in (dict(d_x=None), dict(d_x=x, d_y=h.clone()), dict(d_x=x[:3]), dict(d_x=x, d_w_pre=torch.zeros(63)),
               dict(d_x=x, d_y=h.clone(), d_h_out=h.half()), dict(d_x=x)):
        with pytest.raises(cb.ClbError):
            n.run(h, **kw)
    with pytest.raises(cb.ClbError):  # row pitch not a multiple of 16
        cb.Int8Linear(torch.zeros(8, 60, dtype=torch.int8), torch.zeros(8))
    with pytest.raises(cb.ClbError):
        cb.Int8Linear(torch.zeros(8, 64), torch.zeros(8))
    lin = cb.Int8Linear(torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8))
    with pytest.raises(cb.ClbError):
        lin.run(torch.zeros(4, 64), torch.zeros(4, 8), d_ws=torch.zeros(lin.workspace_bytes(4), dtype=torch.uint8))
    with pytest.raises(cb.ClbError):
        lin.run(torch.zeros(4, 32), torch.zeros(4, 8))


def test_wrappers_refuse_what_is_no_tensor():
    torch = pytest.importorskip("torch")
    r, n = cb.ExpertRoute(64, 6), cb.BlockNorm(64)
    t, ids, w = torch.zeros(4, 64), torch.zeros(4, 6, dtype=torch.int32), torch.zeros(4, 6)
    with pytest.raises(TypeError):
        r.run([[0.0] * 64], ids, w)
    with pytest.raises(TypeError):
        r.run(t, None, w)
    with pytest.raises(TypeError):
        n.run(t, d_y=3, d_h_out=t.clone(), d_x=t.clone())
    with pytest.raises(TypeError):
        cb.Int8Linear(None, w)
    with pytest.raises(cb.ClbError):
        cb.Int8Linear(torch.zeros(8, 64, dtype=torch.int8), None)
    with pytest.raises(cb.ClbError):
        cb.int8_quantize(t, torch.zeros(4, 64, dtype=torch.int8), None)
    with pytest.raises(cb.ClbError):  # no rows of elements
        r.run(t.to_sparse(), ids, w)
    for meta in (t.to("meta"),):  # no storage
        with pytest.raises((cb.ClbError, RuntimeError)):
            r.run(meta, ids, w)
    with pytest.raises(cb.ClbError):  # values of one element: every row the same address
        n.run(torch.zeros(4, 1).expand(4, 64), d_x=t.clone())
    with pytest.raises(cb.ClbError):  # overlapping rows
        n.run(torch.zeros(128).as_strided((4, 64), (16, 1)), d_x=t.clone())


def test_messages_name_the_argument():
    torch = pytest.importorskip("torch")
    r = cb.ExpertRoute(64, 6)
    t, ids, w = torch.zeros(4, 64), torch.zeros(4, 6, dtype=torch.int32), torch.zeros(4, 6)
    for args, word in (((t.double(), ids, w), "logits"), ((t, ids.long(), w), "ids"), ((t, ids, w.half()), "weights"),
                       ((t, ids, w, torch.zeros(63)), "bias"), ((t, ids, w), "CUDA")):
        with pytest.raises(cb.ClbError) as e:
            r.run(*args)
        assert word in str(e.value) and e.value.code == CLB_E_INVALID
