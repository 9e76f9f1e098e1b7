"""The operators around the routed experts of a layer (include/crosslane_b200.h): routing to
experts, the norms with the gated residual step, and the 8-bit integer product.

Each class holds what stays the same from call to call; `run` takes torch tensors on one
CUDA device, launches on that device's current stream (or `stream`) and writes into tensors
of the caller. Rows may lie in a wider buffer: only the last stride has to be 1. Tensors of
another type, shape, stride or device, and outputs that share memory with an input or with one
another (but BlockNorm's d_h_out, which may be d_h), are refused with ClbError.

The tensors are checked and the C entry points called by csrc/torch_call.cpp (a decode step
makes these calls once a layer, with a few microseconds of GPU work each).
"""
import ctypes as C

import torch  # noqa: F401  (the module below is linked against it)

from ._capi import (BlockNormConfigV1, CLB_E_INVALID, ClbError, ErrorV1, Int8LinearConfigV1, RouteConfigV1, check, lib)

try:
    from . import _torch_call as _call
except ImportError as e:
    raise ImportError("crosslane_b200: _torch_call is not built for this Python and torch (run "
                      "`python crosslane_b200/build.py`)") from e

_call.bind(*(C.cast(f, C.c_void_p).value for f in (lib.clb_route_experts_device, lib.clb_block_norm_device,
                                                   lib.clb_int8_quantize_device, lib.clb_int8_linear_device)), ClbError)

SCORES = {"sigmoid": 0, "softmax": 1, "sqrt_softplus": 2}
GROUP_SCORES = {"max": 1, "pair": 2}
GATES = {"none": 0, "channel": 1, "token": 2, "full": 3}


def _refuse(what: str):
    raise ClbError(CLB_E_INVALID, what)


class ExpertRoute:
    """Routing of a layer (clb_route_experts_device): `score` "sigmoid", "softmax" or
    "sqrt_softplus"; the best `top_groups` of `n_groups` groups by "max" or "pair"."""

    def __init__(self, n_experts: int, k: int, *, score: str = "sigmoid", n_groups: int = 1, top_groups: int = 1,
                 group_score: str = "pair", renormalize: bool = True, scale: float = 1.0):
        if score not in SCORES or group_score not in GROUP_SCORES:
            _refuse(f"unknown score {score!r} or group score {group_score!r}")
        self.n_experts, self.k = n_experts, k
        cfg = RouteConfigV1(n_experts=n_experts, k=k, score=SCORES[score], n_groups=n_groups, top_groups=top_groups,
                            group_score=GROUP_SCORES[group_score], renormalize=int(renormalize), scale=scale)
        err = ErrorV1()  # zero tokens: the configuration's own checks
        check(lib.clb_route_experts_device(C.byref(cfg), None, n_experts, None, 0, None, None, None, None, C.byref(err)),
              err)
        self._cfg = bytes(cfg)

    def run(self, d_logits, d_ids, d_w, d_bias=None, d_status=None, stream=None) -> None:
        """d_logits [T][E] (fp32, bf16, fp16) -> d_ids int32 [T][k], d_w fp32 [T][k]; d_bias fp32
        [E]; d_status int32 [1] becomes 1 where a row holds a NaN or +inf."""
        _call.route(self._cfg, d_logits, d_ids, d_w, d_bias, d_status, stream)


class BlockNorm:
    """The residual step between two blocks (clb_block_norm_device):
    h' = residual_scale h + block_scale gate z, z = RMSNorm(y) w_post (`post`) or y;
    x = RMSNorm(h') w_pre (`pre`). gate: "none", "channel" [dim], "token" [T], "full" [T][dim]."""

    def __init__(self, dim: int, *, post: bool = True, pre: bool = True, eps: float = 1e-6, gate: str = "none",
                 gate_sigmoid: bool = False, residual_scale: float = 1.0, block_scale: float = 1.0):
        if gate not in GATES:
            _refuse(f"unknown gate {gate!r}")
        self.dim, self.post, self.pre, self.gate = dim, bool(post), bool(pre), gate
        cfg = BlockNormConfigV1(dim=dim, post=int(post), gate=GATES[gate], gate_sigmoid=int(gate_sigmoid), post_eps=eps,
                                pre_eps=eps, residual_scale=residual_scale, block_scale=block_scale)
        err = ErrorV1()
        check(lib.clb_block_norm_device(C.byref(cfg), 0, None, None, None, None, None, None, None, None, C.byref(err)),
              err)
        self._cfg = bytes(cfg)

    def run(self, d_h, d_y=None, d_gate=None, d_w_post=None, d_w_pre=None, d_h_out=None, d_x=None,
            stream=None) -> None:
        """d_h [T][dim], the block's output d_y, d_h_out (may be d_h) and the next block's input
        d_x; without d_y only x = RMSNorm(h) w_pre. Weights fp32 [dim], None = ones."""
        _call.norm(self._cfg, self.pre, d_h, d_y, d_gate, d_w_post, d_w_pre, d_h_out, d_x, stream)


def int8_quantize(d_x, d_q, d_scale, stream=None) -> None:
    """Rows of d_x [R][K] as int8 d_q [R][K] (row pitch a multiple of 16) with fp32 scales
    d_scale [R] (clb_int8_quantize_device): tokens of an activation, or a weight's channels."""
    _call.quantize(d_x, d_q, d_scale, stream)


class Int8Linear:
    """y = x_scale w_scale (q . w) + bias with int8 weights d_w [N][K] (row pitch a multiple
    of 16) and fp32 d_w_scale [N] (clb_int8_linear_device)."""

    def __init__(self, d_w, d_w_scale, d_bias=None):
        self.n, self.k, ld_w = _call.weights(d_w, d_w_scale, d_bias)
        self.d_w, self.d_w_scale, self.d_bias = d_w, d_w_scale, d_bias
        cfg = Int8LinearConfigV1(n=self.n, k=self.k, ld_w=ld_w, ld_x=(self.k + 15) // 16 * 16, ld_out=self.n)
        err = ErrorV1()
        check(lib.clb_int8_linear_device(C.byref(cfg), None, None, None, 0, None, None, None, None, 0, None, None,
                                         C.byref(err)), err)
        self._cfg = bytes(cfg)

    def workspace_bytes(self, tokens: int) -> int:
        """Bytes of d_ws for `tokens` rows of a floating x."""
        return int(lib.clb_int8_linear_workspace_bytes(tokens, self.k))

    def run(self, d_x, d_out, d_ws=None, d_x_scale=None, d_status=None, stream=None) -> None:
        """d_x [T][K] fp32, bf16 or fp16 (d_ws: uint8 workspace) or int8 with d_x_scale fp32 [T];
        d_out [T][N]. d_status int32 [1] becomes 3 if a wait in the kernel ran out."""
        _call.linear(self._cfg, self.d_w, self.d_w_scale, self.d_bias, d_x, d_out, d_ws, d_x_scale, d_status, stream)
