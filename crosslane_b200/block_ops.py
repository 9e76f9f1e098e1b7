"""The operators around the routed experts of a layer (include/crosslane_b200.h): routing to
experts, the norms with the gated residual step, and the 8-bit integer product.

Each class holds what stays the same from call to call; `run` takes torch tensors on one
CUDA device, launches on that device's current stream (or `stream`) and writes into tensors
of the caller. Rows may lie in a wider buffer: only the last stride has to be 1.
"""
import ctypes as C

import torch

from ._capi import BlockNormConfigV1, CLB_E_INVALID, ClbError, ErrorV1, Int8LinearConfigV1, RouteConfigV1, check, lib

TYPE_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.int8: 3}
SCORES = {"sigmoid": 0, "softmax": 1, "sqrt_softplus": 2}
GROUP_SCORES = {"max": 1, "pair": 2}
GATES = {"none": 0, "channel": 1, "token": 2, "full": 3}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _refuse(what: str):
    raise ClbError(CLB_E_INVALID, what)


def _rows(t, name, types, device, tokens=None, width=None):
    """Row pitch of a [tokens][width] tensor of one of `types` on `device`, its last stride 1."""
    if t.dtype not in types or t.device != device or t.dim() != 2:
        _refuse(f"{name}: a 2-D tensor of {' / '.join(map(str, types))} on {device} is needed")
    n, w = t.shape
    if (tokens is not None and n != tokens) or (width is not None and w != width):
        _refuse(f"{name} is {tuple(t.shape)}, not ({tokens}, {width})")
    if w > 1 and t.stride(1) != 1:
        _refuse(f"{name}: the last stride is {t.stride(1)}, not 1")
    ld = t.stride(0) if n > 1 else max(w, 1)
    if ld < w:
        _refuse(f"{name}: rows overlap (stride {ld}, width {w})")
    return ld


def _vector(t, name, types, device, n):
    if t.dtype not in types or t.device != device or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        _refuse(f"{name}: a contiguous vector of {n} {' / '.join(map(str, types))} on {device} is needed")


def _dense(t, name, dtype, device, shape):
    if t.dtype != dtype or t.device != device or tuple(t.shape) != shape or not t.is_contiguous():
        _refuse(f"{name}: a contiguous {dtype} tensor of shape {shape} on {device} is needed")


class _Call:
    """The device of a call: its current stream, and the device made current if it is not."""

    def __init__(self, device):
        if device.type != "cuda":
            _refuse(f"tensors are on {device}, not on a CUDA device")
        self.index = device.index

    def __call__(self, fn, stream, *args):
        err = ErrorV1()
        if stream is None:
            stream = torch.cuda.current_stream(self.index).cuda_stream
        if torch.cuda.current_device() == self.index:
            rc = fn(*args, stream, C.byref(err))
        else:
            with torch.cuda.device(self.index):
                rc = fn(*args, stream, C.byref(err))
        check(rc, err)


def _ptr(t):
    return None if t is None else t.data_ptr()


class ExpertRoute:
    """Routing of a layer (clb_route_experts_device): `score` "sigmoid", "softmax" or
    "sqrt_softplus"; the best `top_groups` of `n_groups` groups by "max" or "pair"."""

    def __init__(self, n_experts: int, k: int, *, score: str = "sigmoid", n_groups: int = 1, top_groups: int = 1,
                 group_score: str = "pair", renormalize: bool = True, scale: float = 1.0):
        if score not in SCORES or group_score not in GROUP_SCORES:
            _refuse(f"unknown score {score!r} or group score {group_score!r}")
        self.n_experts, self.k = n_experts, k
        self._cfg = RouteConfigV1(n_experts=n_experts, k=k, score=SCORES[score], n_groups=n_groups,
                                  top_groups=top_groups, group_score=GROUP_SCORES[group_score],
                                  renormalize=int(renormalize), scale=scale)
        err = ErrorV1()  # zero tokens: the configuration's own checks
        check(lib.clb_route_experts_device(C.byref(self._cfg), None, n_experts, None, 0, None, None, None, None,
                                           C.byref(err)), err)

    def run(self, d_logits, d_ids, d_w, d_bias=None, d_status=None, stream=None) -> None:
        """d_logits [T][E] (fp32, bf16, fp16) -> d_ids int32 [T][k], d_w fp32 [T][k]; d_bias fp32
        [E]; d_status int32 [1] becomes 1 where a row holds a NaN or +inf."""
        dev = d_logits.device
        ld = _rows(d_logits, "logits", _FLOATS, dev, None, self.n_experts)
        T = d_logits.shape[0]
        _dense(d_ids, "ids", torch.int32, dev, (T, self.k))
        _dense(d_w, "weights", torch.float32, dev, (T, self.k))
        if d_bias is not None:
            _vector(d_bias, "bias", (torch.float32,), dev, self.n_experts)
        if d_status is not None:
            _vector(d_status, "status", (torch.int32,), dev, 1)
        cfg = RouteConfigV1.from_buffer_copy(self._cfg)
        cfg.logits_type = TYPE_CODES[d_logits.dtype]
        _Call(dev)(lib.clb_route_experts_device, stream, C.byref(cfg), _ptr(d_logits), ld, _ptr(d_bias), T, _ptr(d_ids),
                   _ptr(d_w), _ptr(d_status))


class BlockNorm:
    """The residual step between two blocks (clb_block_norm_device):
    h' = residual_scale h + block_scale gate z, z = RMSNorm(y) w_post (`post`) or y;
    x = RMSNorm(h') w_pre (`pre`). gate: "none", "channel" [dim], "token" [T], "full" [T][dim]."""

    def __init__(self, dim: int, *, post: bool = True, pre: bool = True, eps: float = 1e-6, gate: str = "none",
                 gate_sigmoid: bool = False, residual_scale: float = 1.0, block_scale: float = 1.0):
        if gate not in GATES:
            _refuse(f"unknown gate {gate!r}")
        self.dim, self.post, self.pre, self.gate = dim, post, pre, gate
        self._cfg = BlockNormConfigV1(dim=dim, post=int(post), gate=GATES[gate], gate_sigmoid=int(gate_sigmoid),
                                      post_eps=eps, pre_eps=eps, residual_scale=residual_scale,
                                      block_scale=block_scale)
        err = ErrorV1()
        check(lib.clb_block_norm_device(C.byref(self._cfg), 0, None, None, None, None, None, None, None, None,
                                        C.byref(err)), err)

    def run(self, d_h, d_y=None, d_gate=None, d_w_post=None, d_w_pre=None, d_h_out=None, d_x=None,
            stream=None) -> None:
        """d_h [T][dim], the block's output d_y, d_h_out (may be d_h) and the next block's input
        d_x; without d_y only x = RMSNorm(h) w_pre. Weights fp32 [dim], None = ones."""
        dev = d_h.device
        cfg = BlockNormConfigV1.from_buffer_copy(self._cfg)
        cfg.ld_h = _rows(d_h, "h", _FLOATS, dev, None, self.dim)
        T = d_h.shape[0]
        cfg.h_type = TYPE_CODES[d_h.dtype]
        if (d_x is not None) != self.pre:
            _refuse("x goes with the norm before the next block")
        if d_y is not None:
            cfg.ld_y = _rows(d_y, "y", _FLOATS, dev, T, self.dim)
            cfg.y_type = TYPE_CODES[d_y.dtype]
            if d_h_out is None:
                _refuse("h_out goes with y")
            cfg.ld_h_out = _rows(d_h_out, "h_out", (d_h.dtype,), dev, T, self.dim)
        if d_gate is not None:
            if self.gate == "full":
                cfg.ld_gate = _rows(d_gate, "gate", _FLOATS, dev, T, self.dim)
            else:
                _vector(d_gate, "gate", _FLOATS, dev, self.dim if self.gate == "channel" else T)
            cfg.gate_type = TYPE_CODES[d_gate.dtype]
        for w, name in ((d_w_post, "w_post"), (d_w_pre, "w_pre")):
            if w is not None:
                _vector(w, name, (torch.float32,), dev, self.dim)
        if d_x is not None:
            cfg.ld_x = _rows(d_x, "x", _FLOATS, dev, T, self.dim)
            cfg.x_type = TYPE_CODES[d_x.dtype]
        _Call(dev)(lib.clb_block_norm_device, stream, C.byref(cfg), T, _ptr(d_h), _ptr(d_y), _ptr(d_gate),
                   _ptr(d_w_post), _ptr(d_w_pre), _ptr(d_h_out), _ptr(d_x))


def int8_quantize(d_x, d_q, d_scale, stream=None) -> None:
    """Rows of d_x [R][K] as int8 d_q [R][K] (row pitch a multiple of 16) with fp32 scales
    d_scale [R] (clb_int8_quantize_device): tokens of an activation, or a weight's channels."""
    dev = d_x.device
    ld_x = _rows(d_x, "x", _FLOATS, dev)
    rows, k = d_x.shape
    ld_q = _rows(d_q, "q", (torch.int8,), dev, rows, k)
    _vector(d_scale, "scale", (torch.float32,), dev, rows)
    if rows == 1:
        ld_q = (k + 15) // 16 * 16
    _Call(dev)(lib.clb_int8_quantize_device, stream, TYPE_CODES[d_x.dtype], _ptr(d_x), ld_x, rows, k, _ptr(d_q), ld_q,
               _ptr(d_scale))


class Int8Linear:
    """y = x_scale w_scale (q . w) + bias with int8 weights d_w [N][K] (row pitch a multiple
    of 16) and fp32 d_w_scale [N] (clb_int8_linear_device)."""

    def __init__(self, d_w, d_w_scale, d_bias=None):
        dev = d_w.device
        ld = _rows(d_w, "w", (torch.int8,), dev)
        self.n, self.k = d_w.shape
        _vector(d_w_scale, "w_scale", (torch.float32,), dev, self.n)
        if d_bias is not None:
            _vector(d_bias, "bias", (torch.float32,), dev, self.n)
        if self.n == 1:
            ld = (self.k + 15) // 16 * 16
        self.d_w, self.d_w_scale, self.d_bias = d_w, d_w_scale, d_bias
        self._cfg = Int8LinearConfigV1(n=self.n, k=self.k, ld_w=ld, ld_x=(self.k + 15) // 16 * 16, ld_out=self.n)
        err = ErrorV1()
        check(lib.clb_int8_linear_device(C.byref(self._cfg), None, None, None, 0, None, None, None, None, 0, None, None,
                                         C.byref(err)), err)

    def workspace_bytes(self, tokens: int) -> int:
        """Bytes of d_ws for `tokens` rows of a floating x."""
        return int(lib.clb_int8_linear_workspace_bytes(tokens, self.k))

    def run(self, d_x, d_out, d_ws=None, d_x_scale=None, d_status=None, stream=None) -> None:
        """d_x [T][K] fp32, bf16 or fp16 (d_ws: uint8 workspace) or int8 with d_x_scale fp32 [T];
        d_out [T][N]. d_status int32 [1] becomes 3 if a wait in the kernel ran out."""
        dev = self.d_w.device
        cfg = Int8LinearConfigV1.from_buffer_copy(self._cfg)
        cfg.ld_x = _rows(d_x, "x", _FLOATS + (torch.int8,), dev, None, self.k)
        T = d_x.shape[0]
        if T == 1 and d_x.dtype == torch.int8:
            cfg.ld_x = (self.k + 15) // 16 * 16
        cfg.ld_out = _rows(d_out, "out", _FLOATS, dev, T, self.n)
        cfg.x_type, cfg.out_type = TYPE_CODES[d_x.dtype], TYPE_CODES[d_out.dtype]
        if d_x_scale is not None:
            _vector(d_x_scale, "x_scale", (torch.float32,), dev, T)
        if d_ws is not None:
            _vector(d_ws, "workspace", (torch.uint8,), dev, d_ws.numel())
        if d_status is not None:
            _vector(d_status, "status", (torch.int32,), dev, 1)
        _Call(dev)(lib.clb_int8_linear_device, stream, C.byref(cfg), _ptr(self.d_w), _ptr(self.d_w_scale),
                   _ptr(self.d_bias), T, _ptr(d_x), _ptr(d_x_scale), _ptr(d_out), _ptr(d_ws),
                   0 if d_ws is None else d_ws.numel(), _ptr(d_status))
