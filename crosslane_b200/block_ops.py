"""The operators around the routed experts of a layer (include/crosslane_b200.h): routing to
experts, the norms with the gated residual step, and the 8-bit integer product.

Each class holds what stays the same from call to call; `run` takes torch tensors on one
CUDA device, launches on that device's current stream (or `stream`) and writes into tensors
of the caller. Rows may lie in a wider buffer: only the last stride has to be 1.

A decode step makes these calls once a layer with a few microseconds of GPU work each, so the
checks read every attribute of a tensor once, and the C structs of a tensor layout are kept
(by types and pitches).
"""
import ctypes as C
import threading

import torch

from ._capi import BlockNormConfigV1, CLB_E_INVALID, ClbError, ErrorV1, Int8LinearConfigV1, RouteConfigV1, check, lib

SCORES = {"sigmoid": 0, "softmax": 1, "sqrt_softplus": 2}
GROUP_SCORES = {"max": 1, "pair": 2}
GATES = {"none": 0, "channel": 1, "token": 2, "full": 3}
# element types of each argument: torch dtype -> CLB_F32 / CLB_BF16 / CLB_F16 / CLB_I8
_FLOAT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ANY = {**_FLOAT, torch.int8: 3}
_F32, _I8, _I32, _U8 = {torch.float32: 0}, {torch.int8: 3}, {torch.int32: 4}, {torch.uint8: 5}
_LAYOUTS = 64  # kept C structs of an operator

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _Local(threading.local):
    def __init__(self):
        self.err = ErrorV1()
        self.ref = C.byref(self.err)


_local = _Local()


def _refuse(what: str):
    raise ClbError(CLB_E_INVALID, what)


def _names(types):
    return " / ".join(str(t).replace("torch.", "") for t in types)


def _device(t):
    index = t.get_device()
    if index < 0:
        _refuse(f"tensors are on {t.device}, not on a CUDA device")
    return index


def _rows(t, name, types, index, tokens, width):
    """(type, row pitch) of a [tokens][width] tensor on CUDA device `index` (-1: not checked, any
    count for tokens or width -1), its last stride 1."""
    code = types.get(t.dtype)
    shape = t.shape
    if code is None or len(shape) != 2 or (t.get_device() != index and index >= 0):
        _refuse(f"{name}: a 2-D tensor of {_names(types)} on the operator's device is needed")
    n, w = shape
    if (n != tokens and tokens >= 0) or (w != width and width >= 0):
        _refuse(f"{name} is {tuple(shape)}, not ({tokens}, {width})")
    ld, step = t.stride()
    if step != 1 and w > 1:
        _refuse(f"{name}: the last stride is {step}, not 1")
    if n <= 1:
        ld = w  # the pitch of a single row is never used
    elif ld < w:
        _refuse(f"{name}: rows overlap (stride {ld}, width {w})")
    return code, ld


def _vector(t, name, types, index, n):
    code = types.get(t.dtype)
    shape = t.shape
    if code is None or len(shape) != 1 or shape[0] != n or (t.get_device() != index and index >= 0) or \
            (n > 1 and t.stride(0) != 1):
        _refuse(f"{name}: a contiguous vector of {n} {_names(types)} on the operator's device is needed")
    return code


def _dense(t, name, types, index, tokens, width):
    if _rows(t, name, types, index, tokens, width)[1] != width:
        _refuse(f"{name}: a contiguous tensor is needed")


def _call(fn, index, stream, *args):
    """fn(*args, stream, err) with device `index` current."""
    if stream is None:
        stream = _raw_stream(index)
    if _current_device() == index:
        rc = fn(*args, stream, _local.ref)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream, _local.ref)
    if rc:
        check(rc, _local.err)


def _layout(kept, key, make):
    if len(kept) >= _LAYOUTS:
        kept.clear()
    cfg = make()
    kept[key] = ref = C.byref(cfg)
    return ref


class ExpertRoute:
    """Routing of a layer (clb_route_experts_device): `score` "sigmoid", "softmax" or
    "sqrt_softplus"; the best `top_groups` of `n_groups` groups by "max" or "pair"."""

    def __init__(self, n_experts: int, k: int, *, score: str = "sigmoid", n_groups: int = 1, top_groups: int = 1,
                 group_score: str = "pair", renormalize: bool = True, scale: float = 1.0):
        if score not in SCORES or group_score not in GROUP_SCORES:
            _refuse(f"unknown score {score!r} or group score {group_score!r}")
        self.n_experts, self.k = n_experts, k
        self._cfgs = tuple(C.byref(RouteConfigV1(n_experts=n_experts, k=k, score=SCORES[score], n_groups=n_groups,
                                                 top_groups=top_groups, group_score=GROUP_SCORES[group_score],
                                                 renormalize=int(renormalize), scale=scale, logits_type=t))
                           for t in sorted(_FLOAT.values()))
        err = ErrorV1()  # zero tokens: the configuration's own checks
        check(lib.clb_route_experts_device(self._cfgs[0], None, n_experts, None, 0, None, None, None, None,
                                           C.byref(err)), err)

    def run(self, d_logits, d_ids, d_w, d_bias=None, d_status=None, stream=None) -> None:
        """d_logits [T][E] (fp32, bf16, fp16) -> d_ids int32 [T][k], d_w fp32 [T][k]; d_bias fp32
        [E]; d_status int32 [1] becomes 1 where a row holds a NaN or +inf."""
        E = self.n_experts
        kind, ld = _rows(d_logits, "logits", _FLOAT, -1, -1, E)
        index = _device(d_logits)
        T = d_logits.shape[0]
        _dense(d_ids, "ids", _I32, index, T, self.k)
        _dense(d_w, "weights", _F32, index, T, self.k)
        bias = status = None
        if d_bias is not None:
            _vector(d_bias, "bias", _F32, index, E)
            bias = d_bias.data_ptr()
        if d_status is not None:
            _vector(d_status, "status", _I32, index, 1)
            status = d_status.data_ptr()
        _call(lib.clb_route_experts_device, index, stream, self._cfgs[kind], d_logits.data_ptr(), ld, bias, T,
              d_ids.data_ptr(), d_w.data_ptr(), status)


class BlockNorm:
    """The residual step between two blocks (clb_block_norm_device):
    h' = residual_scale h + block_scale gate z, z = RMSNorm(y) w_post (`post`) or y;
    x = RMSNorm(h') w_pre (`pre`). gate: "none", "channel" [dim], "token" [T], "full" [T][dim]."""

    def __init__(self, dim: int, *, post: bool = True, pre: bool = True, eps: float = 1e-6, gate: str = "none",
                 gate_sigmoid: bool = False, residual_scale: float = 1.0, block_scale: float = 1.0):
        if gate not in GATES:
            _refuse(f"unknown gate {gate!r}")
        self.dim, self.post, self.pre, self.gate = dim, post, pre, gate
        self._fixed = dict(dim=dim, post=int(post), gate=GATES[gate], gate_sigmoid=int(gate_sigmoid), post_eps=eps,
                           pre_eps=eps, residual_scale=residual_scale, block_scale=block_scale)
        self._kept = {}
        err = ErrorV1()
        check(lib.clb_block_norm_device(C.byref(BlockNormConfigV1(**self._fixed)), 0, None, None, None, None, None, None,
                                        None, None, C.byref(err)), err)

    def run(self, d_h, d_y=None, d_gate=None, d_w_post=None, d_w_pre=None, d_h_out=None, d_x=None,
            stream=None) -> None:
        """d_h [T][dim], the block's output d_y, d_h_out (may be d_h) and the next block's input
        d_x; without d_y only x = RMSNorm(h) w_pre. Weights fp32 [dim], None = ones."""
        dim = self.dim
        h_type, ld_h = _rows(d_h, "h", _FLOAT, -1, -1, dim)
        index = _device(d_h)
        T = d_h.shape[0]
        y_type = x_type = g_type = ld_y = ld_x = ld_g = ld_o = 0
        y = gate = w_post = w_pre = h_out = x = None
        if (d_x is not None) != self.pre:
            _refuse("x goes with the norm before the next block")
        if d_y is not None:
            y_type, ld_y = _rows(d_y, "y", _FLOAT, index, T, dim)
            if d_h_out is None:
                _refuse("h_out goes with y")
            o_type, ld_o = _rows(d_h_out, "h_out", _FLOAT, index, T, dim)
            if o_type != h_type:
                _refuse("h_out has another type than h")
            y, h_out = d_y.data_ptr(), d_h_out.data_ptr()
        elif d_h_out is not None:
            _refuse("h_out goes with y")
        if d_gate is not None:
            if self.gate == "full":
                g_type, ld_g = _rows(d_gate, "gate", _FLOAT, index, T, dim)
            else:
                g_type = _vector(d_gate, "gate", _FLOAT, index, dim if self.gate == "channel" else T)
            gate = d_gate.data_ptr()
        if d_w_post is not None:
            _vector(d_w_post, "w_post", _F32, index, dim)
            w_post = d_w_post.data_ptr()
        if d_w_pre is not None:
            _vector(d_w_pre, "w_pre", _F32, index, dim)
            w_pre = d_w_pre.data_ptr()
        if d_x is not None:
            x_type, ld_x = _rows(d_x, "x", _FLOAT, index, T, dim)
            x = d_x.data_ptr()
        key = (h_type, y_type, g_type, x_type, ld_h, ld_y, ld_g, ld_o, ld_x)
        cfg = self._kept.get(key) or _layout(self._kept, key, lambda: BlockNormConfigV1(
            h_type=h_type, y_type=y_type, gate_type=g_type, x_type=x_type, ld_h=ld_h, ld_y=ld_y, ld_gate=ld_g,
            ld_h_out=ld_o, ld_x=ld_x, **self._fixed))
        _call(lib.clb_block_norm_device, index, stream, cfg, T, d_h.data_ptr(), y, gate, w_post, w_pre, h_out, x)


def _pitch16(rows, k, ld):
    """The pitch of int8 rows; that of a single row is never used."""
    return (k + 15) // 16 * 16 if rows <= 1 else ld


def int8_quantize(d_x, d_q, d_scale, stream=None) -> None:
    """Rows of d_x [R][K] as int8 d_q [R][K] (row pitch a multiple of 16) with fp32 scales
    d_scale [R] (clb_int8_quantize_device): tokens of an activation, or a weight's channels."""
    kind, ld_x = _rows(d_x, "x", _FLOAT, -1, -1, -1)
    index = _device(d_x)
    rows, k = d_x.shape
    ld_q = _pitch16(rows, k, _rows(d_q, "q", _I8, index, rows, k)[1])
    _vector(d_scale, "scale", _F32, index, rows)
    _call(lib.clb_int8_quantize_device, index, stream, kind, d_x.data_ptr(), ld_x, rows, k, d_q.data_ptr(), ld_q,
          d_scale.data_ptr())


class Int8Linear:
    """y = x_scale w_scale (q . w) + bias with int8 weights d_w [N][K] (row pitch a multiple
    of 16) and fp32 d_w_scale [N] (clb_int8_linear_device)."""

    def __init__(self, d_w, d_w_scale, d_bias=None):
        self._index = d_w.get_device()
        ld = _rows(d_w, "w", _I8, -1, -1, -1)[1]
        self.n, self.k = d_w.shape
        for t, name in ((d_w_scale, "w_scale"), (d_bias, "bias")):
            if t is not None:
                if t.get_device() != self._index:
                    _refuse(f"{name} is on another device than the weights")
                _vector(t, name, _F32, self._index, self.n)
        self.d_w, self.d_w_scale, self.d_bias = d_w, d_w_scale, d_bias
        self._fixed = dict(n=self.n, k=self.k, ld_w=_pitch16(self.n, self.k, ld))
        self._kept = {}
        err = ErrorV1()
        cfg = Int8LinearConfigV1(ld_x=(self.k + 15) // 16 * 16, ld_out=self.n, **self._fixed)
        check(lib.clb_int8_linear_device(C.byref(cfg), None, None, None, 0, None, None, None, None, 0, None, None,
                                         C.byref(err)), err)

    def workspace_bytes(self, tokens: int) -> int:
        """Bytes of d_ws for `tokens` rows of a floating x."""
        return int(lib.clb_int8_linear_workspace_bytes(tokens, self.k))

    def run(self, d_x, d_out, d_ws=None, d_x_scale=None, d_status=None, stream=None) -> None:
        """d_x [T][K] fp32, bf16 or fp16 (d_ws: uint8 workspace) or int8 with d_x_scale fp32 [T];
        d_out [T][N]. d_status int32 [1] becomes 3 if a wait in the kernel ran out."""
        index = self._index
        if index < 0:
            _refuse(f"the weights are on {self.d_w.device}, not on a CUDA device")
        x_type, ld_x = _rows(d_x, "x", _ANY, index, -1, self.k)
        T = d_x.shape[0]
        if x_type == 3:
            ld_x = _pitch16(T, self.k, ld_x)
        out_type, ld_out = _rows(d_out, "out", _FLOAT, index, T, self.n)
        scale = ws = status = None
        ws_bytes = 0
        if d_x_scale is not None:
            _vector(d_x_scale, "x_scale", _F32, index, T)
            scale = d_x_scale.data_ptr()
        if d_ws is not None:
            ws_bytes = d_ws.numel()
            _vector(d_ws, "workspace", _U8, index, ws_bytes)
            ws = d_ws.data_ptr()
        if d_status is not None:
            _vector(d_status, "status", _I32, index, 1)
            status = d_status.data_ptr()
        key = (x_type, out_type, ld_x, ld_out)
        cfg = self._kept.get(key) or _layout(self._kept, key, lambda: Int8LinearConfigV1(
            x_type=x_type, out_type=out_type, ld_x=ld_x, ld_out=ld_out, **self._fixed))
        _call(lib.clb_int8_linear_device, index, stream, cfg, self.d_w.data_ptr(), self.d_w_scale.data_ptr(),
              None if self.d_bias is None else self.d_bias.data_ptr(), T, d_x.data_ptr(), scale, d_out.data_ptr(), ws,
              ws_bytes, status)
