"""nk.py — Python binding of libnk's C ABI (include/nk.h) over ctypes.

Device memory, streams and process groups come from PyTorch; every compute
call goes through libnk.so (sm_100a kernels).  There is no CPU path: when
libnk.so is missing or no GPU is present, calls raise.

The wrappers mirror the reference's kernel-wrapper API
(nemotron-kernels/src/{gemm,quantize,moe_routing}.rs): same argument order
and the same error variants, raised as NkError with the variant's payload.
"""
from __future__ import annotations

import array
import ctypes
import os
from dataclasses import dataclass

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("NK_LIB_PATH") or os.path.join(_HERE, "libnk.so")

# status codes (nk.h)
OK, INVALID_SHAPE, LENGTH_MISMATCH, INVALID_PARAMS, INT4_OUT_OF_RANGE = 0, 1, 2, 3, 4
NON_FINITE_INPUT, INVALID_ROW_COUNT, UNSUPPORTED, DEVICE_ERROR, TIMEOUT = 5, 6, 7, 8, 9
WORKSPACE_TOO_SMALL, INVALID_DELTA_T, EMPTY_INPUT, NEGATIVE_EPSILON = 10, 11, 12, 13
HEAD_COUNT_MISMATCH, INVALID_SCALE, NO_VALID_TARGETS, ZERO_PARTITION = 14, 15, 16, 17
TOKEN_OUT_OF_RANGE, PAGE_OUT_OF_RANGE = 18, 19
STATUS_NAMES = {
    0: "Ok", 1: "InvalidShape", 2: "LengthMismatch", 3: "InvalidParams",
    4: "Int4OutOfRange", 5: "NonFiniteInput", 6: "InvalidRowCount", 7: "Unsupported",
    8: "DeviceError", 9: "Timeout", 10: "WorkspaceTooSmall", 11: "InvalidDeltaT",
    12: "EmptyInput", 13: "NegativeEpsilon", 14: "HeadCountMismatch", 15: "InvalidScale",
    16: "NoValidAttentionTargets", 17: "ZeroPartition", 18: "TokenOutOfRange",
    19: "PageOutOfRange",
}
F32, BF16 = 0, 1
EPI_RELU2 = 1
ROUTE_SIGMOID, ROUTE_SOFTMAX, ROUTE_SIGMOID_RENORM = 0, 1, 2
W_BF16, W_INT8_ROW, W_INT4_AFFINE = 0, 1, 2

_c = ctypes
_sz = _c.c_size_t
_i64 = _c.c_int64
_i32 = _c.c_int32
_u32 = _c.c_uint32
_p = _c.c_void_p
_f = _c.c_float


class NkErrorInfo(_c.Structure):
    _fields_ = [
        ("code", _c.c_int32),
        ("argument", _c.c_char * 32),
        ("expected", _c.c_uint64),
        ("actual", _c.c_uint64),
        ("index", _c.c_uint64),
        ("value", _c.c_float),
        ("byte_value", _c.c_uint32),
        ("message", _c.c_char * 256),
    ]


class NkMoeLayer(_c.Structure):
    _fields_ = [
        ("hidden", _i64), ("experts", _i64), ("top_k", _i64), ("inter", _i64),
        ("shared_inter", _i64), ("route_mode", _i32), ("weight_kind", _i32),
        ("router_w3", _p), ("router_b", _p),
        ("up_w", _p), ("up_scale", _p), ("up_b", _p),
        ("down_w", _p), ("down_scale", _p), ("down_b", _p),
        ("shared_up_w", _p), ("shared_up_scale", _p), ("shared_up_b", _p),
        ("shared_down_w", _p), ("shared_down_scale", _p), ("shared_down_b", _p),
        ("up_zero_point", _p), ("down_zero_point", _p),
        ("shared_up_zero_point", _p), ("shared_down_zero_point", _p),
        ("router_norms", _p),
    ]


class NkConvArgs(_c.Structure):
    _fields_ = [
        ("batch", _i64), ("seq", _i64), ("channels", _i64), ("kernel_size", _i64),
        ("x", _p), ("ld_x", _i64), ("weights", _p), ("prefix", _p), ("silu", _i32),
        ("y", _p), ("ld_y", _i64), ("state_out", _p), ("f32_accumulate", _i32),
    ]


class NkScanArgs(_c.Structure):
    _fields_ = [
        ("batch", _i64), ("seq", _i64), ("channels", _i64), ("states", _i64),
        ("x", _p), ("ld_x", _i64),
        ("dt", _p), ("ld_dt", _i64), ("dt_group", _i32),
        ("a", _p), ("a_group", _i32), ("a_per_state", _i32),
        ("b", _p), ("c", _p), ("ld_bc", _i64), ("bc_group", _i32),
        ("d", _p), ("d_group", _i32),
        ("initial_state", _p),
        ("delta_bias", _f), ("softplus", _i32),
        ("y", _p), ("ld_y", _i64),
        ("final_state", _p),
        ("check_delta_t", _i32),
    ]


class NkKvPages(_c.Structure):
    _fields_ = [
        ("layers", _i64), ("pages", _i64), ("kv_heads", _i64), ("page_size", _i64),
        ("head_dim", _i64), ("k", _p), ("v", _p), ("k_min", _p), ("k_max", _p),
        ("table", _p), ("table_rows", _i64), ("table_ld", _i64),
    ]


class NkKvBatch(_c.Structure):
    _fields_ = [
        ("seqs", _i64), ("tokens", _i64), ("start", _p), ("kv_len", _p), ("rows", _p),
        ("max_new", _i64), ("max_kv", _i64),
    ]


class NkKvCompactArgs(_c.Structure):
    _fields_ = [
        ("seqs", _i64), ("rows", _p), ("kv_len", _p), ("base", _p), ("keep", _p),
        ("keep_ld", _i64), ("n_keep", _p), ("max_keep", _i64), ("dst_table", _p),
        ("dst_ld", _i64), ("new_len", _p),
    ]


class NkPagedAttentionArgs(_c.Structure):
    _fields_ = [
        ("q", _p), ("ld_q", _i64), ("q_heads", _i64), ("tree_mask", _p), ("blocks", _p),
        ("max_blocks", _i64), ("has_scale", _i32), ("scale", _f), ("out", _p),
        ("out_dtype", _i32),
    ]


class NkError(Exception):
    """A libnk status other than NK_OK, with the matching Rust variant's payload."""

    def __init__(self, info: NkErrorInfo):
        self.code = int(info.code)
        self.variant = STATUS_NAMES.get(self.code, str(self.code))
        self.argument = info.argument.decode()
        self.expected = int(info.expected)
        self.actual = int(info.actual)
        self.index = int(info.index)
        self.value = float(info.value)
        self.byte_value = int(info.byte_value)
        self.message = info.message.decode(errors="replace")
        super().__init__(f"{self.variant}: {self.message}")


# name -> (restype, argtypes)
_SIGS = {
    "nk_last_error": (_i32, [_p]),
    "nk_version": (_i32, []),
    "nk_device_status": (_i32, [_p]),
    "nk_gemm_f32": (_i32, [_p, _sz, _p, _sz, _p, _sz, _sz, _sz, _sz, _p]),
    "nk_gemm_bf16": (_i32, [_p, _i32, _p, _p, _p, _i32, _i64, _i64, _i64, _i32, _p]),
    "nk_gemm_w8row": (_i32, [_p, _i32, _p, _p, _p, _p, _i32, _i64, _i64, _i64, _i32, _p]),
    "nk_gemm_w8row_f32_static": (_i32, [_p, _p, _p, _p, _p, _i32, _i64, _i64, _i64, _i32, _p]),
    "nk_gemm_w4a": (_i32, [_p, _i32, _p, _sz, _f, _u32, _p, _p, _i32, _i64, _i64, _i64, _i32, _p]),
    "nk_gemm_workspace_bytes": (_i32, [_i32, _i32, _i64, _i64, _i64, _p]),
    "nk_gemm_bf16_ws": (_i32, [_p, _i32, _p, _p, _p, _i32, _i64, _i64, _i64, _i32, _p, _sz, _p]),
    "nk_gemm_w8row_ws": (_i32, [_p, _i32, _p, _p, _p, _p, _i32, _i64, _i64, _i64, _i32, _p, _sz,
                                _p]),
    "nk_gemm_w4a_ws": (_i32, [_p, _i32, _p, _sz, _f, _u32, _p, _p, _i32, _i64, _i64, _i64, _i32,
                              _p, _sz, _p]),
    "nk_scratch_release": (_i32, [_p]),
    "nk_ep_handle_bytes": (_sz, []),
    "nk_ep_create": (_i32, [_i32, _i32, _i64, _i64, _i64, _i64, _i64, _p, _p]),
    "nk_ep_connect": (_i32, [_p, _p]),
    "nk_moe_forward_ep_workspace_bytes": (_i32, [_p, _p, _p, _i64, _p]),
    "nk_moe_forward_ep": (_i32, [_p, _p, _p, _p, _i64, _p, _i32, _p, _p, _p, _sz, _p]),
    "nk_ep_barrier": (_i32, [_p, _p]),
    "nk_ep_received_rows": (_i32, [_p, _p]),
    "nk_ep_destroy": (_i32, [_p]),
    "nk_pack_int4": (_i32, [_p, _sz, _p, _sz, _p]),
    "nk_unpack_int4": (_i32, [_p, _sz, _sz, _p, _sz, _p]),
    "nk_quantize_int4": (_i32, [_p, _sz, _f, _u32, _p, _sz, _p]),
    "nk_int4_kn_to_nk": (_i32, [_p, _i64, _i64, _i64, _p, _p]),
    "nk_router_norms": (_i32, [_p, _i64, _i64, _p, _p]),
    "nk_dequantize_int4": (_i32, [_p, _sz, _sz, _f, _u32, _p, _sz, _p]),
    "nk_validate_int4_params": (_i32, [_f, _u32]),
    "nk_quantize_int8_row": (_i32, [_p, _i64, _i64, _p, _p, _p]),
    "nk_moe_route": (_i32, [_p, _sz, _sz, _sz, _sz, _i32, _p, _sz, _p, _sz, _p]),
    "nk_moe_plan": (_i32, [_p, _i64, _i64, _i64, _p, _p, _p, _p, _p]),
    "nk_router_split": (_i32, [_p, _i64, _i64, _p, _p]),
    "nk_linear_pack_kn": (_i32, [_p, _i64, _i64, _p, _p]),
    "nk_moe_workspace_bytes": (_i32, [_p, _i64, _p]),
    "nk_moe_forward": (_i32, [_p, _p, _i64, _p, _i32, _p, _p, _p, _sz, _p]),
    "nk_selftest_wait_timeout": (_i32, [_p]),
    "nk_moe_pipeline_create": (_i32, [_p, _i64, _i32, _p, _p, _p, _p]),
    "nk_moe_pipeline_submit": (_i32, [_p, _p, _i64, _p, _p]),
    "nk_moe_pipeline_wait": (_i32, [_p]),
    "nk_moe_pipeline_destroy": (_i32, [_p]),
    "nk_moe_dispatch_workspace_bytes": (_i32, [_p, _i64, _p]),
    "nk_moe_dispatch": (_i32, [_p, _p, _i64, _p, _p, _p, _p, _p, _p, _p, _sz, _p]),
    "nk_moe_experts_workspace_bytes": (_i32, [_p, _i64, _i32, _p]),
    "nk_moe_experts": (_i32, [_p, _p, _i64, _p, _p, _i32, _p, _p, _sz, _p]),
    "nk_moe_shared": (_i32, [_p, _p, _i64, _p, _p, _p]),
    "nk_moe_combine": (_i32, [_p, _p, _p, _p, _i64, _i64, _i64, _p, _i32, _p]),
    "nk_ipc_alloc": (_i32, [_sz, _p, _p]),
    "nk_ipc_open": (_i32, [_p, _p]),
    "nk_ipc_close": (_i32, [_p]),
    "nk_ipc_free": (_i32, [_p]),
    "nk_ep_plan": (_i32, [_p, _i32, _i32, _i32, _p, _p, _p, _p, _p, _p]),
    "nk_ep_dispatch": (_i32, [_p, _i64, _i64, _i32, _p, _p, _p, _p, _i32, _p, _p]),
    "nk_ep_return": (_i32, [_p, _i64, _i32, _i32, _p, _p, _p, _p, _p]),
    "nk_ep_plan_phased": (_i32, [_p, _i32, _i32, _i32, _i32, _i64, _p, _p, _p, _p, _p, _p]),
    "nk_ep_dispatch_phase": (_i32, [_p, _i64, _i64, _i32, _p, _p, _p, _p, _i32, _i32, _i32, _p,
                                    _p]),
    "nk_ep_return_segments": (_i32, [_p, _i64, _i32, _i32, _i32, _i32, _p, _p, _p, _p, _p]),
    "nk_conv1d": (_i32, [_p, _sz, _p, _sz, _i64, _i64, _i64, _p, _sz, _p]),
    "nk_conv1d_ex": (_i32, [_p, _p]),
    "nk_selective_scan": (_i32, [_p, _sz, _p, _sz, _p, _sz, _p, _sz, _p, _sz, _p, _sz, _p, _sz,
                                 _f, _i32, _i64, _i64, _i64, _p, _sz, _p, _sz, _p]),
    "nk_selective_scan_ex": (_i32, [_p, _p]),
    "nk_rms_norm": (_i32, [_p, _sz, _p, _sz, _p, _sz, _f, _p, _sz, _p]),
    "nk_rms_norm_rows": (_i32, [_p, _i64, _i64, _i64, _p, _sz, _p, _i64, _f, _p, _i64, _i32,
                                _p]),
    "nk_row_sumsq": (_i32, [_p, _i64, _i64, _i64, _p, _p]),
    "nk_rms_norm_rows_presummed": (_i32, [_p, _i64, _i64, _i64, _p, _sz, _p, _i64, _p, _i64,
                                          _f, _p, _i64, _i32, _p]),
    "nk_attention_f32": (_i32, [_p, _sz, _p, _sz, _p, _sz, _i64, _i64, _i64, _i64, _i64, _i64,
                                _i32, _i64, _i32, _f, _p, _sz, _p]),
    "nk_kv_append": (_i32, [_p, _p, _i64, _i64, _i64, _i64, _i64, _i64, _p, _p, _p]),
    "nk_attention_workspace_bytes": (_i32, [_i64, _i64, _i64, _i64, _i64, _i64, _i64, _p]),
    "nk_attention_gqa": (_i32, [_p, _p, _p, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _i32,
                                _i64, _i32, _f, _p, _i32, _p, _sz, _p]),
    "nk_attention_check": (_i32, [_p, _p, _p]),
    "nk_embedding_lookup": (_i32, [_p, _i32, _sz, _p, _i64, _i64, _i64, _p, _i32, _sz, _i32, _p]),
    "nk_add_rms_norm_rows": (_i32, [_p, _p, _i64, _i64, _p, _sz, _f, _p, _p, _i32, _p]),
    "nk_argmax_rows": (_i32, [_p, _i32, _i64, _i64, _i64, _p, _p]),
    "nk_kv_pages_append": (_i32, [_p, _i64, _p, _p, _i64, _p, _i64, _p]),
    "nk_kv_pages_copy": (_i32, [_p, _p, _p, _i64, _p]),
    "nk_kv_table_write": (_i32, [_p, _i64, _p, _p, _i64, _p]),
    "nk_kv_pages_compact": (_i32, [_p, _p, _p]),
    "nk_attention_paged_workspace_bytes": (_i32, [_p, _p, _p, _p]),
    "nk_attention_paged": (_i32, [_p, _i64, _p, _p, _p, _sz, _p]),
    "nk_kv_block_select_workspace_bytes": (_i32, [_p, _p, _p]),
    "nk_kv_block_select": (_i32, [_p, _i64, _p, _p, _i64, _i64, _i64, _i64, _i64, _p, _p, _sz,
                                  _p]),
    "nk_set_stage_timing": (_i32, [_i32]),
    "nk_moe_stage_times": (_i32, [_p, _i32, _p]),
}
MOE_STAGES = ("router", "route_plan", "gather", "up_proj", "down_proj", "shared_expert",
              "combine")


def set_stage_timing(enable: bool) -> None:
    call("nk_set_stage_timing", 1 if enable else 0)


def moe_stage_times() -> dict:
    """Per-stage milliseconds of this thread's last nk_moe_forward (see nk.h)."""
    arr = (ctypes.c_float * len(MOE_STAGES))()
    n = ctypes.c_int32(0)
    call("nk_moe_stage_times", arr, len(MOE_STAGES), ctypes.byref(n))
    return {MOE_STAGES[i]: float(arr[i]) for i in range(n.value)}

_lib = None


def lib() -> ctypes.CDLL:
    """Loads libnk.so (built in-tree by `make -C nemotron-cutile-rs_b200`)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"libnk.so not built: {LIB_PATH} (run make -C {_HERE})")
        h = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(h, name)
            fn.restype = res
            fn.argtypes = args
        _lib = h
    return _lib


def last_error() -> NkErrorInfo:
    info = NkErrorInfo()
    lib().nk_last_error(ctypes.byref(info))
    return info


def check(status: int) -> None:
    if status != OK:
        raise NkError(last_error())


def call(name: str, *args) -> None:
    """Calls an nk_* entry point and raises NkError on a non-OK status."""
    status = getattr(_lib or lib(), name)(*args)
    if status != OK:
        raise NkError(last_error())


# ----------------------------------------------------------------- torch glue
def ptr(t) -> int | None:
    """Device address of a tensor (None for None)."""
    return None if t is None else t.data_ptr()


def stream_ptr(stream=None) -> int:
    import torch

    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("libnk entry points take device tensors")


# ------------------------------------------------------------ kernel wrappers
def gemm_f32(lhs, rhs, m: int, k: int, n: int, out=None, stream=None):
    """nemotron_kernels::gemm::gemm / gemm_into (gemm.rs:318-363)."""
    import torch

    _require_cuda(lhs, rhs, out)
    if out is None:
        out = torch.empty(m * n if m * n > 0 else 1, dtype=torch.float32, device=lhs.device)
        out_len = m * n
    else:
        out_len = out.numel()
    call("nk_gemm_f32", ptr(lhs), lhs.numel(), ptr(rhs), rhs.numel(), ptr(out), out_len,
         m, k, n, stream_ptr(stream))
    return out


def gemm_workspace_bytes(kind: str, x_dtype, m: int, k: int, n: int) -> int:
    """nk_gemm_workspace_bytes: scratch the *_ws projections need for this shape."""
    import torch

    wk = {"bf16": W_BF16, "int8": W_INT8_ROW, "int4": W_INT4_AFFINE}[kind]
    b = ctypes.c_size_t(0)
    call("nk_gemm_workspace_bytes", wk, F32 if x_dtype == torch.float32 else BF16, m, k, n,
         ctypes.byref(b))
    return b.value


def gemm(x, w, *, kind: str = "bf16", bias=None, scales=None, scale: float = 1.0,
         zero_point: int = 0, n: int | None = None, out_dtype=None, relu2: bool = False,
         stream=None, workspace=None):
    """Projection Y[M,N] = X[M,K]·Wᵀ (+bias) (relu2) — LinearProjection::project_into.

    kind: "bf16" (w bf16 [N,K]), "int8" (w int8 [N,K], scales f32 [N]),
    "int4" (w uint8 packed reference layout [K,N], scale/zero_point).
    workspace: optional uint8 device tensor of >= gemm_workspace_bytes (the
    *_ws entry points); by default the library's per-stream scratch.
    """
    import torch

    _require_cuda(x, w, bias, scales)
    m, k = x.shape
    x_dtype = F32 if x.dtype == torch.float32 else BF16
    if kind == "int4":
        assert n is not None
    else:
        n = w.shape[0]
    out_dtype = out_dtype or torch.float32
    y = torch.empty((m, n), dtype=out_dtype, device=x.device)
    y_dtype = F32 if out_dtype == torch.float32 else BF16
    flags = EPI_RELU2 if relu2 else 0
    s = stream_ptr(stream)
    if workspace is not None:
        wsp, wsn = ptr(workspace), workspace.numel()
        if kind == "bf16":
            call("nk_gemm_bf16_ws", ptr(x), x_dtype, ptr(w), ptr(bias), ptr(y), y_dtype, m, k, n,
                 flags, wsp, wsn, s)
        elif kind == "int8":
            call("nk_gemm_w8row_ws", ptr(x), x_dtype, ptr(w), ptr(scales), ptr(bias), ptr(y),
                 y_dtype, m, k, n, flags, wsp, wsn, s)
        elif kind == "int4":
            call("nk_gemm_w4a_ws", ptr(x), x_dtype, ptr(w), w.numel(), float(scale),
                 int(zero_point), ptr(bias), ptr(y), y_dtype, m, k, n, flags, wsp, wsn, s)
        else:
            raise ValueError(kind)
        return y
    if kind == "bf16":
        call("nk_gemm_bf16", ptr(x), x_dtype, ptr(w), ptr(bias), ptr(y), y_dtype, m, k, n, flags, s)
    elif kind == "int8":
        call("nk_gemm_w8row", ptr(x), x_dtype, ptr(w), ptr(scales), ptr(bias), ptr(y), y_dtype,
             m, k, n, flags, s)
    elif kind == "int4":
        call("nk_gemm_w4a", ptr(x), x_dtype, ptr(w), w.numel(), float(scale), int(zero_point),
             ptr(bias), ptr(y), y_dtype, m, k, n, flags, s)
    else:
        raise ValueError(kind)
    return y


def moe_route(scores, tokens: int, experts: int, top_k: int, mode: int = ROUTE_SIGMOID,
              stream=None):
    """moe_routing::moe_route / moe_route_softmax (moe_routing.rs:499-532)."""
    import torch

    _require_cuda(scores)
    dev = scores.device
    n = max(tokens * top_k, 1)  # placeholder storage when the batch is empty
    idx = torch.empty(n, dtype=torch.int32, device=dev)
    w = torch.empty(n, dtype=torch.float32, device=dev)
    call("nk_moe_route", ptr(scores), scores.numel(), tokens, experts, top_k, mode, ptr(idx),
         tokens * top_k, ptr(w), tokens * top_k, stream_ptr(stream))
    return idx[: tokens * top_k], w[: tokens * top_k]


def moe_plan(indices, tokens: int, top_k: int, experts: int, stream=None):
    import torch

    dev = indices.device
    slots = tokens * top_k
    counts = torch.empty(experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(max(slots, 1), dtype=torch.int32, device=dev)
    pos = torch.empty(max(slots, 1), dtype=torch.int32, device=dev)
    call("nk_moe_plan", ptr(indices), tokens, top_k, experts, ptr(counts), ptr(offsets),
         ptr(perm), ptr(pos), stream_ptr(stream))
    return counts, offsets, perm[:slots], pos[:slots]


def quantize_int8_row(w, stream=None):
    import torch

    n, k = w.shape
    q = torch.empty((n, k), dtype=torch.int8, device=w.device)
    s = torch.empty(n, dtype=torch.float32, device=w.device)
    call("nk_quantize_int8_row", ptr(w), n, k, ptr(q), ptr(s), stream_ptr(stream))
    return q, s


def quantize_int4_experts(w, zero_point: int = 8, stream=None):
    """Expert weights w [E, N, K] (output-major, any float dtype) in the
    reference's INT4-affine format, one per-tensor (scale, zero_point) per
    expert: scale = max|W_e| / 7 as the benchmark configurations state, codes
    from nk_quantize_int4 (quantize.rs:131-144) on W_eᵀ in the reference's
    [K, N] = [input_dim, output_dim] layout.  Returns (codes [E, N, K/2] uint8
    feature-major for NK_W_INT4_AFFINE, scales f32 [E], zero points uint8 [E],
    reference packed bytes [E, ceil(K*N/2)])."""
    import torch

    e, n, k = w.shape
    wf = w.float()
    scales = (wf.abs().amax(dim=(1, 2)) / 7.0).to(torch.float32)
    kn_len = (k * n + 1) // 2
    packed = torch.empty((e, kn_len), dtype=torch.uint8, device=w.device)
    sc = scales.cpu().tolist()
    for i in range(e):
        t = wf[i].t().contiguous()  # [K, N]
        call("nk_quantize_int4", ptr(t), k * n, float(sc[i]), zero_point, ptr(packed[i]), kn_len,
             stream_ptr(stream))
    codes = torch.empty((e, n, k // 2), dtype=torch.uint8, device=w.device)
    call("nk_int4_kn_to_nk", ptr(packed), e, k, n, ptr(codes), stream_ptr(stream))
    zps = torch.full((e,), zero_point, dtype=torch.uint8, device=w.device)
    return codes, scales, zps, packed


def router_split(w, stream=None):
    import torch

    e, h = w.shape
    hp = (h + 63) // 64 * 64
    w3 = torch.empty((e, 3 * hp), dtype=torch.bfloat16, device=w.device)
    call("nk_router_split", ptr(w), e, h, ptr(w3), stream_ptr(stream))
    return w3


@dataclass
class MoeWeights:
    """Device tensors of one MoE layer in libnk's layouts (see nk_moe_layer)."""
    hidden: int
    experts: int
    top_k: int
    inter: int
    shared_inter: int
    route_mode: int
    weight_kind: int
    router_w3: object
    router_b: object = None
    up_w: object = None
    up_scale: object = None
    up_b: object = None
    down_w: object = None
    down_scale: object = None
    down_b: object = None
    shared_up_w: object = None
    shared_up_scale: object = None
    shared_up_b: object = None
    shared_down_w: object = None
    shared_down_scale: object = None
    shared_down_b: object = None
    up_zero_point: object = None          # INT4_AFFINE: uint8 [E]
    down_zero_point: object = None
    shared_up_zero_point: object = None   # uint8 [1]
    shared_down_zero_point: object = None
    router_norms: object = None           # f32 [2E] (nk_router_norms), or computed per call

    def struct(self) -> NkMoeLayer:
        s = NkMoeLayer()
        for f in ("hidden", "experts", "top_k", "inter", "shared_inter", "route_mode",
                  "weight_kind"):
            setattr(s, f, getattr(self, f))
        for f in ("router_w3", "router_b", "up_w", "up_scale", "up_b", "down_w", "down_scale",
                  "down_b", "shared_up_w", "shared_up_scale", "shared_up_b", "shared_down_w",
                  "shared_down_scale", "shared_down_b", "up_zero_point", "down_zero_point",
                  "shared_up_zero_point", "shared_down_zero_point", "router_norms"):
            setattr(s, f, ptr(getattr(self, f)))
        return s


def ensure_router_norms(weights: MoeWeights) -> None:
    """Fills weights.router_norms once (nk_router_norms) so that forwards skip it."""
    import torch

    if weights.router_norms is None and weights.router_w3 is not None:
        weights.router_norms = torch.empty(2 * weights.experts, dtype=torch.float32,
                                           device=weights.router_w3.device)
        call("nk_router_norms", ptr(weights.router_w3), weights.experts, weights.hidden,
             ptr(weights.router_norms), stream_ptr())


class MoeLayer:
    """Device MoE layer: MoeLayer::forward_into (nemotron-nn/src/moe.rs:154-249)."""

    def __init__(self, weights: MoeWeights):
        ensure_router_norms(weights)
        self.weights = weights
        self._struct = weights.struct()
        self._ws = None

    def workspace_bytes(self, tokens: int) -> int:
        b = ctypes.c_size_t(0)
        call("nk_moe_workspace_bytes", ctypes.byref(self._struct), tokens, ctypes.byref(b))
        return b.value

    def forward(self, x, out=None, out_dtype=None, indices=None, weights=None, stream=None,
                workspace=None):
        """workspace: an optional uint8 device buffer shared by several layers
        (grown in place, as a one-element list [tensor]); by default the layer
        keeps its own."""
        import torch

        t = x.shape[0]
        need = self.workspace_bytes(t)
        if workspace is not None:
            if workspace[0] is None or workspace[0].numel() < need:
                workspace[0] = None
                workspace[0] = torch.empty(need, dtype=torch.uint8, device=x.device)
            self._ws = workspace[0]
        elif self._ws is None or self._ws.numel() < need:
            self._ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        if out is None:
            out = torch.empty((t, self.weights.hidden), dtype=out_dtype or torch.float32,
                              device=x.device)
        od = F32 if out.dtype == torch.float32 else BF16
        call("nk_moe_forward", ctypes.byref(self._struct), ptr(x), t, ptr(out), od, ptr(indices),
             ptr(weights), ptr(self._ws), self._ws.numel(), stream_ptr(stream))
        return out


class MoePipeline:
    """Host-buffer MoE forwards (nk_moe_pipeline_*): submit(x_host, out_host)
    copies x in, runs the layer and copies out, overlapping the copies of
    adjacent submissions with the forward in between.  x_host / out_host are
    CPU tensors (pinned for the copies to overlap); results are valid after
    wait().  streams: optional (h2d, compute, d2h) torch.cuda.Stream triple."""

    def __init__(self, layer: MoeLayer, max_tokens: int, out_dtype=None, streams=None):
        import torch

        self.layer = layer  # keeps the weights (and the layer struct) alive
        self.streams = streams
        od = BF16 if out_dtype == torch.bfloat16 else F32
        self.out_dtype = torch.bfloat16 if od == BF16 else torch.float32
        self.max_tokens = max_tokens
        h = ctypes.c_void_p()
        sp = [None, None, None] if streams is None else [s.cuda_stream for s in streams]
        call("nk_moe_pipeline_create", ctypes.byref(layer._struct), max_tokens, od, *sp,
             ctypes.byref(h))
        self._h = h

    def submit(self, x_host, out_host, indices_host=None):
        import torch

        for t in (x_host, out_host, indices_host):
            if t is not None and (t.is_cuda or not t.is_contiguous()):
                raise ValueError("host tensors must be contiguous CPU tensors")
        hidden, top_k = self.layer.weights.hidden, self.layer.weights.top_k
        if x_host.dtype != torch.bfloat16 or x_host.dim() != 2 or x_host.shape[1] != hidden:
            raise ValueError(f"x_host must be bf16 [tokens, {hidden}]")
        tokens = x_host.shape[0]
        if out_host.dtype != self.out_dtype or out_host.numel() < tokens * hidden:
            raise ValueError("out_host must hold tokens x hidden values of the pipeline's dtype")
        if indices_host is not None and (indices_host.dtype != torch.int32 or
                                         indices_host.numel() < tokens * top_k):
            raise ValueError("indices_host must hold tokens x top_k int32 values")
        call("nk_moe_pipeline_submit", self._h, x_host.data_ptr(), tokens, out_host.data_ptr(),
             None if indices_host is None else indices_host.data_ptr())

    def wait(self):
        call("nk_moe_pipeline_wait", self._h)

    def close(self):
        if self._h:
            call("nk_moe_pipeline_destroy", self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def device_status(stream=None) -> None:
    call("nk_device_status", stream_ptr(stream))


# ------------------------------------------------------------- Mamba2 glue
def _numel(t) -> int:
    return 0 if t is None else t.numel()


def conv1d(inp, weights, seq: int, channels: int, kernel_size: int, out=None, stream=None):
    """depthwise_causal_conv1d (conv1d.rs:78-124, 325-345) on device f32 tensors."""
    import torch

    _require_cuda(inp, weights, out)
    if out is None:
        out = torch.empty(max(seq * channels, 1), dtype=torch.float32, device=inp.device)
        out_len = seq * channels
    else:
        out_len = out.numel()
    call("nk_conv1d", ptr(inp), inp.numel(), ptr(weights), weights.numel(), seq, channels,
         kernel_size, ptr(out), out_len, stream_ptr(stream))
    return out[:out_len]


def conv1d_ex(x, weights, batch: int, seq: int, channels: int, kernel_size: int, *,
              ld_x=None, prefix=None, silu=False, y=None, ld_y=None, state_out=None,
              f32_accumulate=False, stream=None):
    """Batched causal conv with conv-cache history and fused SiLU (mamba2.rs:276-312)."""
    import torch

    _require_cuda(x, weights, prefix, y, state_out)
    if y is None:
        y = torch.empty(batch * seq, channels, dtype=torch.float32, device=x.device)
        ld_y = channels
    a = NkConvArgs(batch, seq, channels, kernel_size, ptr(x), ld_x or channels, ptr(weights),
                   ptr(prefix), 1 if silu else 0, ptr(y), ld_y or channels, ptr(state_out),
                   1 if f32_accumulate else 0)
    call("nk_conv1d_ex", ctypes.byref(a), stream_ptr(stream))
    return y


def selective_scan(inp, delta_t, a, b, c, seq: int, channels: int, states: int, *, d=None,
                   initial_state=None, delta_bias: float = 0.0, softplus: bool = False,
                   out=None, final_state=None, stream=None):
    """selective_scan (ssm.rs:123-175, 614-624).  Returns (values, final_state)."""
    import torch

    _require_cuda(inp, delta_t, a, b, c, d, initial_state, out, final_state)
    dev = inp.device
    ol = seq * channels if out is None else out.numel()
    fl = channels * states if final_state is None else final_state.numel()
    if out is None:
        out = torch.empty(max(ol, 1), dtype=torch.float32, device=dev)
    if final_state is None:
        final_state = torch.empty(max(fl, 1), dtype=torch.float32, device=dev)
    call("nk_selective_scan", ptr(inp), inp.numel(), ptr(delta_t), delta_t.numel(), ptr(a),
         a.numel(), ptr(b), b.numel(), ptr(c), c.numel(), ptr(d), _numel(d),
         ptr(initial_state), _numel(initial_state), delta_bias, 1 if softplus else 0, seq,
         channels, states, ptr(out), ol, ptr(final_state), fl, stream_ptr(stream))
    return out[:ol], final_state[:fl]


def selective_scan_ex(args: NkScanArgs, stream=None) -> None:
    """Strided / shared-parameter scan (nk_selective_scan_ex); args hold device pointers."""
    call("nk_selective_scan_ex", ctypes.byref(args), stream_ptr(stream))


def rms_norm(inp, weight, epsilon: float, gate=None, out=None, stream=None):
    """rms_norm_into_host / gated_rms_norm_into_host (rms_norm.rs:64-106) on device."""
    import torch

    _require_cuda(inp, weight, gate, out)
    n = inp.numel()
    ol = n if out is None else out.numel()
    if out is None:
        out = torch.empty(max(n, 1), dtype=torch.float32, device=inp.device)
    call("nk_rms_norm", ptr(inp), n, ptr(weight), weight.numel(), ptr(gate), _numel(gate),
         epsilon, ptr(out), ol, stream_ptr(stream))
    return out[:ol]


def rms_norm_rows(x, weight, epsilon: float, gate=None, out_dtype: int = F32, out=None,
                  stream=None):
    """Row-wise (gated) RMSNorm (rms_norm.rs:291-360, mamba2.rs:567-586); x is [rows, width]
    (row stride taken from the tensor), gate likewise or None."""
    import torch

    _require_cuda(x, weight, gate, out)
    rows, width = x.shape
    if out is None:
        out = torch.empty(rows, width, device=x.device,
                          dtype=torch.bfloat16 if out_dtype == BF16 else torch.float32)
    call("nk_rms_norm_rows", ptr(x), rows, width, x.stride(0), ptr(weight), weight.numel(),
         ptr(gate), gate.stride(0) if gate is not None else 0, epsilon, ptr(out),
         out.stride(0), out_dtype, stream_ptr(stream))
    return out


def row_sumsq(x, out=None, stream=None):
    """f64 sum of squares of each row of x [rows, width] (nk_row_sumsq)."""
    import torch

    _require_cuda(x, out)
    rows, width = x.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.float64, device=x.device)
    call("nk_row_sumsq", ptr(x), rows, width, x.stride(0), ptr(out), stream_ptr(stream))
    return out


def rms_norm_rows_presummed(x, weight, epsilon: float, sumsq, total_width: int, gate=None,
                            out_dtype: int = F32, out=None, stream=None):
    """Row-wise (gated) RMSNorm of the local columns of rows split over ranks;
    sumsq [rows] f64 holds the full rows' sums of squares."""
    import torch

    _require_cuda(x, weight, gate, sumsq, out)
    rows, width = x.shape
    if out is None:
        out = torch.empty(rows, width, device=x.device,
                          dtype=torch.bfloat16 if out_dtype == BF16 else torch.float32)
    call("nk_rms_norm_rows_presummed", ptr(x), rows, width, x.stride(0), ptr(weight),
         weight.numel(), ptr(gate), gate.stride(0) if gate is not None else 0, ptr(sumsq),
         total_width, epsilon, ptr(out), out.stride(0), out_dtype, stream_ptr(stream))
    return out


# ------------------------------------------------------------ attention core
def attention_f32(q, k, v, batch, q_seq, kv_seq, q_heads, kv_heads, head_dim, *, causal=False,
                  q_offset=0, scale=None, out=None, stream=None):
    """scaled_dot_product_attention (attention.rs:204-302) on f32 [B, S, H, d] device tensors."""
    import torch

    _require_cuda(q, k, v, out)
    n = batch * q_seq * q_heads * head_dim
    ol = n if out is None else out.numel()
    if out is None:
        out = torch.empty(max(n, 1), dtype=torch.float32, device=q.device)
    call("nk_attention_f32", ptr(q), q.numel(), ptr(k), k.numel(), ptr(v), v.numel(), batch,
         q_seq, kv_seq, q_heads, kv_heads, head_dim, 1 if causal else 0, q_offset,
         0 if scale is None else 1, 0.0 if scale is None else scale, ptr(out), ol,
         stream_ptr(stream))
    return out[:ol]


class KvCache:
    """The serving KV cache: K [B, Hkv, max_len, d] and V transposed
    [B, Hkv, d, max_len], bf16, zero-initialised (nk_kv_append)."""

    def __init__(self, batch, kv_heads, head_dim, max_len, device="cuda"):
        import torch

        self.batch, self.kv_heads, self.head_dim, self.max_len = batch, kv_heads, head_dim, max_len
        self.k = torch.zeros(batch, kv_heads, max_len, head_dim, dtype=torch.bfloat16,
                             device=device)
        self.vt = torch.zeros(batch, kv_heads, head_dim, max_len, dtype=torch.bfloat16,
                              device=device)
        self.length = 0

    def append(self, k_new, v_new, seq, stream=None):
        """k_new / v_new bf16 [batch*seq, kv_heads*head_dim] at positions length.. ."""
        _require_cuda(k_new, v_new)
        call("nk_kv_append", ptr(k_new), ptr(v_new), self.batch, seq, self.kv_heads,
             self.head_dim, self.length, self.max_len, ptr(self.k), ptr(self.vt),
             stream_ptr(stream))
        self.length += seq


def attention_gqa(q, cache: KvCache, q_seq, q_heads, *, causal=True, q_offset=None, scale=None,
                  out_dtype=BF16, out=None, workspace=None, stream=None):
    """Grouped-query attention of q bf16 [B*q_seq, q_heads*d] over the cache's
    first `cache.length` positions (nk_attention_gqa).  q_offset defaults to
    cache.length - q_seq (the queries are the last q_seq positions)."""
    import torch

    _require_cuda(q, out, workspace)
    B, Hkv, d, L = cache.batch, cache.kv_heads, cache.head_dim, cache.length
    if q_offset is None:
        q_offset = L - q_seq
    need = ctypes.c_size_t(0)
    call("nk_attention_workspace_bytes", B, q_seq, L, cache.max_len, q_heads, Hkv, d,
         ctypes.byref(need))
    if workspace is None or workspace.numel() < need.value:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
    if out is None:
        out = torch.empty(B * q_seq, q_heads * d, device=q.device,
                          dtype=torch.float32 if out_dtype == F32 else torch.bfloat16)
    call("nk_attention_gqa", ptr(q), ptr(cache.k), ptr(cache.vt), B, q_seq, L, cache.max_len,
         q_heads, Hkv, d, 1 if causal else 0, q_offset, 0 if scale is None else 1,
         0.0 if scale is None else scale, ptr(out), out_dtype, ptr(workspace),
         workspace.numel(), stream_ptr(stream))
    return out, workspace


def attention_check(workspace, stream=None) -> int:
    """First output row without a finite score in the last nk_attention_gqa, or -1."""
    r = ctypes.c_int64(0)
    call("nk_attention_check", ptr(workspace), ctypes.byref(r), stream_ptr(stream))
    return r.value


# ------------------------------------------------------------- paged KV cache
# The wrappers below are called several times a decode step, where the GPU work
# of a call is a few microseconds: they look at each property of a tensor once
# and leave the wording of refusals to the slow path.  With stream= the inputs
# must be ready on that stream; results may be read on the current one once it
# waits for the other.
def _is(t, dtype, dim, device) -> bool:
    return t.dtype is dtype and t.dim() == dim and t.device == device and \
        (t.is_contiguous() or t.stride(-1) == 1)


def _expect(t, name, dtype, dim, device=None):
    """A device tensor of the given type and rank whose last dimension is dense."""
    if t.dtype != dtype or t.dim() != dim:
        raise TypeError(f"{name} must be {dtype} with {dim} dimensions, got {t.dtype} "
                        f"{tuple(t.shape)}")
    if not t.is_cuda:
        raise RuntimeError("libnk entry points take device tensors")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, the pages on {device}")
    if t.numel() and t.stride(-1) != 1:
        raise ValueError(f"{name} must be dense in its last dimension")


def _expect_ints(t, name, n, device):
    import torch

    if not _is(t, torch.int32, 1, device):
        _expect(t, name, torch.int32, 1, device)
    if t.numel() != n:
        raise ValueError(f"{name} must hold {n} values, got {t.numel()}")


def _call_on(device, name, *args) -> None:
    """call() with the tensors' device current: libnk launches on the current one."""
    import torch

    if device.index == torch._C._cuda_getDevice():
        call(name, *args)
    else:
        with torch.cuda.device(device):
            call(name, *args)


def _stream_of(device, stream) -> int:
    """The stream to launch on: the given one or the device's current one."""
    import torch

    return stream.cuda_stream if stream is not None else \
        torch._C._cuda_getCurrentRawStream(device.index)


def _empty(shape, dtype, device, stream, result=True):
    """New device memory for a call on `stream`.  On an explicit stream it comes
    from that stream's memory: the current stream's may have been freed by work
    that is still queued there.  result: the caller reads it on the current
    stream, so it is not given out again before that stream's work is done with
    it either."""
    import torch

    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        t = torch.empty(shape, dtype=dtype, device=device)
    if result:
        t.record_stream(torch.cuda.current_stream(device))
    return t


def _bytes_of(workspace, device) -> int:
    """Size of a workspace that the caller may have given."""
    import torch

    if workspace.dtype is not torch.uint8 or workspace.device != device or \
            not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous uint8 memory of {device}")
    return workspace.numel()


class KvPages:
    """A pool of KV pages and the table that strings them into sequences
    (nk_kv_pages): k, v bf16 [layers, pages, kv_heads, page_size, head_dim],
    table int32 [sequences, blocks]; k_min, k_max bf16 [layers, pages,
    kv_heads, head_dim] hold the channel bounds of each page's keys, which
    kv_block_select reads (optional).  nk_paged.PagedKvCache manages one."""

    def __init__(self, k, v, table, *, k_min=None, k_max=None):
        import torch

        _expect(k, "k", torch.bfloat16, 5)
        dev = k.device
        _expect(v, "v", torch.bfloat16, 5, dev)
        _expect(table, "table", torch.int32, 2, dev)
        if v.shape != k.shape or not (k.is_contiguous() and v.is_contiguous()):
            raise ValueError("k and v must be contiguous and of one shape")
        if (k_min is None) != (k_max is None):
            raise ValueError("k_min and k_max go together")
        for t, name in ((k_min, "k_min"), (k_max, "k_max")):
            if t is not None:
                _expect(t, name, torch.bfloat16, 4, dev)
                if t.shape != k.shape[:3] + k.shape[4:] or not t.is_contiguous():
                    raise ValueError(f"{name} must be contiguous [layers, pages, kv_heads, "
                                     "head_dim]")
        self.k, self.v, self.table, self.k_min, self.k_max = k, v, table, k_min, k_max
        self.layers, self.num_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.device = dev
        # The library takes a row for table_ld entries long.  Where rows lie further
        # apart, max_kv holds a batch to the columns that are there.
        ld = table.stride(0) if table.shape[0] > 1 else table.shape[1]
        self._apart = ld > table.shape[1]
        self._struct = NkKvPages(*k.shape, ptr(k), ptr(v), ptr(k_min), ptr(k_max), ptr(table),
                                 table.shape[0], ld)
        self._ref = ctypes.byref(self._struct)
        self._bytes = {}  # bounds of an attention call -> its workspace bytes

    def batch(self, start, kv_len, tokens, max_new, max_kv=None, rows=None) -> NkKvBatch:
        """The ragged batch of one step (nk_kv_batch): start int32 [n + 1],
        kv_len int32 [n], rows int32 [n] or None on the pages' device; max_kv
        defaults to what the table can hold, max_new None is all tokens, or
        max_kv where a sequence cannot hold them all."""
        n = kv_len.numel()
        _expect_ints(start, "start", n + 1, self.device)
        _expect_ints(kv_len, "kv_len", n, self.device)
        if rows is not None:
            _expect_ints(rows, "rows", n, self.device)
        if max_kv is None or self._apart:
            held = self.table.shape[1] * self.page_size
            max_kv = held if max_kv is None else min(max_kv, held)
        if max_new is None:
            max_new = min(tokens, max_kv)
        return NkKvBatch(n, tokens, start.data_ptr(), kv_len.data_ptr(),
                         None if rows is None else rows.data_ptr(), max_new, max_kv)

    def _attend_bytes(self, b, q_heads, max_blocks):
        """Workspace bytes of an attention call: its bounds alone decide."""
        key = (b.tokens, b.seqs, q_heads, b.max_new, b.max_kv, max_blocks)
        size = self._bytes.get(key)
        if size is None:
            # of the pointers only whether they are there is read
            a = NkPagedAttentionArgs(None, q_heads * self.head_dim, q_heads, None,
                                     16 if max_blocks else None, max_blocks, 0, 0.0, None, BF16)
            size = self._ask_bytes(key, "nk_attention_paged_workspace_bytes", b, ctypes.byref(a))
        return size

    def _select_bytes(self, b):
        """Workspace bytes of kv_block_select."""
        key = (b.tokens, b.seqs, b.max_new, b.max_kv)
        size = self._bytes.get(key)
        if size is None:
            size = self._ask_bytes(key, "nk_kv_block_select_workspace_bytes", b)
        return size

    def _ask_bytes(self, key, name, b, *args):
        need = ctypes.c_size_t(0)
        _call_on(self.device, name, self._ref, ctypes.byref(b), *args, ctypes.byref(need))
        if len(self._bytes) > 4096:  # lengths that grow with each step
            self._bytes.clear()
        size = self._bytes[key] = need.value
        return size

    def _queries(self, q, q_heads):
        import torch

        if not _is(q, torch.bfloat16, 2, self.device):
            _expect(q, "q", torch.bfloat16, 2, self.device)
        tokens, width = q.shape
        if width != q_heads * self.head_dim:
            raise ValueError(f"q must be [tokens, {q_heads * self.head_dim}]")
        return tokens, (q.stride(0) if tokens > 1 else width)


def kv_pages_append(pages: KvPages, k_new, v_new, start, kv_len, *, max_new, max_kv=None,
                    rows=None, layer: int = 0, stream=None) -> None:
    """Stores new keys and values (bf16 [tokens, kv_heads * head_dim], any row
    stride that is a multiple of 8) at the last positions of their sequences
    (nk_kv_pages_append).  max_kv defaults to what the table can hold."""
    import torch

    width = pages.kv_heads * pages.head_dim
    tokens = k_new.shape[0]
    for t, name in ((k_new, "k_new"), (v_new, "v_new")):
        if not _is(t, torch.bfloat16, 2, pages.device):
            _expect(t, name, torch.bfloat16, 2, pages.device)
        if t.shape != (tokens, width):
            raise ValueError(f"{name} must be [tokens, {width}]")
    b = pages.batch(start, kv_len, tokens, max_new, max_kv, rows)
    ld_k, ld_v = (k_new.stride(0), v_new.stride(0)) if tokens > 1 else (width, width)
    _call_on(pages.device, "nk_kv_pages_append", pages._ref, layer, ctypes.byref(b),
             k_new.data_ptr(), ld_k, v_new.data_ptr(), ld_v, _stream_of(pages.device, stream))


# Host arrays go to the library as bytes, which ctypes passes by address: an
# array's own address takes 2.5 us to ask for.
def _host_ints(a, dtype):
    import numpy as np

    if isinstance(a, (list, tuple, range)):  # an array.array takes whole numbers that fit
        try:
            return np.frombuffer(array.array("i" if dtype is np.int32 else "q", a), dtype)
        except TypeError:
            raise ValueError(f"not a sequence of whole numbers: {a}") from None
    a = np.asarray(a)
    if a.dtype != dtype and a.size:
        b = a.astype(dtype)
        if a.dtype.kind not in "iu" or (b != a).any():
            raise ValueError(f"{a.dtype} values do not fit {np.dtype(dtype)}")
        a = b
    return np.ascontiguousarray(a, dtype=dtype)


def kv_pages_copy(pages: KvPages, src, dst, stream=None) -> None:
    """Page dst[i] becomes a copy of page src[i] in every layer
    (nk_kv_pages_copy); src, dst are host sequences of page ids."""
    import numpy as np

    s, d = _host_ints(src, np.int32), _host_ints(dst, np.int32)
    if s.size != d.size:
        raise ValueError("src and dst must have one length")
    _call_on(pages.device, "nk_kv_pages_copy", pages._ref, s.tobytes(), d.tobytes(), s.size,
             _stream_of(pages.device, stream))


def kv_table_write(dst, values, offsets=None, stream=None) -> None:
    """dst.view(-1)[offsets[i]] = values[i] (nk_kv_table_write; offsets None:
    the first len(values) entries); dst is a contiguous int32 device tensor,
    values and offsets are host sequences."""
    import numpy as np
    import torch

    if dst.dtype != torch.int32 or not dst.is_contiguous():
        raise TypeError("dst must be a contiguous int32 tensor")
    _require_cuda(dst)
    v = _host_ints(values, np.int32)
    o = None if offsets is None else _host_ints(offsets, np.int64)
    if o is not None and o.size != v.size:
        raise ValueError("offsets and values must have one length")
    _call_on(dst.device, "nk_kv_table_write", ptr(dst), dst.numel(),
             None if o is None else o.tobytes(), v.tobytes(), v.size,
             _stream_of(dst.device, stream))


def _rows_together(table, stream):
    """A page table that the call only reads, its rows one behind the other: the
    device checks lengths against the distance of rows."""
    import torch

    if table.shape[0] <= 1 or table.stride(0) == table.shape[1]:
        return table
    with torch.cuda.stream(stream):  # None: the current one
        return table.contiguous()


def kv_pages_compact(pages: KvPages, kv_len, base, keep, n_keep, *, rows=None, dst_table=None,
                     new_len=None, stream=None):
    """Token base[b] + keep[b, i] of sequence b moves to position base[b] + i
    (nk_kv_pages_compact), in place or into the pages of dst_table; all
    arguments int32 on the device, keep [n, max_keep] strictly ascending.
    Returns the new lengths base + n_keep, in new_len where it is given (not an
    array that the call reads)."""
    import torch

    n, dev = kv_len.numel(), pages.device
    for t, name in ((kv_len, "kv_len"), (base, "base"), (n_keep, "n_keep")):
        _expect_ints(t, name, n, dev)
    if rows is not None:
        _expect_ints(rows, "rows", n, dev)
    _expect(keep, "keep", torch.int32, 2, dev)
    if keep.shape[0] != n:
        raise ValueError("keep must have a row for each sequence")
    dst, dst_ld = None, 0
    if dst_table is not None:
        _expect(dst_table, "dst_table", torch.int32, 2, dev)
        if dst_table.shape[0] != n:
            raise ValueError("dst_table must have a row for each sequence")
        if dst_table.shape[1] == 0:  # its address would be none: in place
            raise ValueError("dst_table must have a column")
        dst_table = _rows_together(dst_table, stream)
        dst, dst_ld = dst_table.data_ptr(), dst_table.shape[1]
    if new_len is None:
        new_len = _empty(n, torch.int32, dev, stream)
    else:
        _expect_ints(new_len, "new_len", n, dev)
    width = keep.shape[1]
    a = NkKvCompactArgs(n, ptr(rows), kv_len.data_ptr(), base.data_ptr(), keep.data_ptr(),
                        keep.stride(0) if n > 1 else width, n_keep.data_ptr(), width, dst, dst_ld,
                        new_len.data_ptr())
    kv = pages._ref
    if pages._apart:
        table = _rows_together(pages.table, stream)
        kv = NkKvPages.from_buffer_copy(pages._struct)
        kv.table, kv.table_ld = table.data_ptr(), table.shape[1]
        kv = ctypes.byref(kv)
    _call_on(dev, "nk_kv_pages_compact", kv, ctypes.byref(a), _stream_of(dev, stream))
    return new_len


def _attend(pages, q, ld_q, b, q_heads, tree_mask, blocks, layer, scale, out_dtype, out,
            workspace, stream):
    """attention_paged behind its checks of q and the batch b."""
    import torch

    dev, tokens = pages.device, q.shape[0]
    max_blocks = 0
    if tree_mask is not None:
        _expect(tree_mask, "tree_mask", torch.int64, 1, dev)
        if tree_mask.numel() != tokens:
            raise ValueError("tree_mask must hold a word for each token")
    if blocks is not None:
        _expect(blocks, "blocks", torch.int32, 3, dev)
        if blocks.shape[:2] != (tokens, pages.kv_heads) or not blocks.is_contiguous():
            raise ValueError("blocks must be contiguous [tokens, kv_heads, n]")
        if blocks.shape[2] == 0:  # its address would be none: attention without lists
            raise ValueError("blocks must hold an entry a list")
        max_blocks = blocks.shape[2] if tokens else 0
    if out is None:
        if stream is None and out_dtype == BF16 and ld_q == q.shape[1]:
            out = torch.empty_like(q)
        else:
            out = _empty(q.shape, torch.float32 if out_dtype == F32 else torch.bfloat16, dev,
                         stream)
        code = out_dtype
    elif out.shape != q.shape or not out.is_contiguous() or out.device != dev:
        raise ValueError("out must be contiguous, of q's shape and on its device")
    else:
        code = _dtype_code(out)
    a = NkPagedAttentionArgs(q.data_ptr(), ld_q, q_heads, ptr(tree_mask), ptr(blocks), max_blocks,
                             0 if scale is None else 1, 0.0 if scale is None else scale,
                             out.data_ptr(), code)
    br, ar = ctypes.byref(b), ctypes.byref(a)
    if workspace is None:
        size = pages._attend_bytes(b, q_heads, max_blocks)
        if size:
            workspace = _empty(size, torch.uint8, dev, stream, result=False)
    else:
        size = _bytes_of(workspace, dev)
    _call_on(dev, "nk_attention_paged", pages._ref, layer, br, ar, ptr(workspace), size,
             _stream_of(dev, stream))
    return out


def attention_paged(q, pages: KvPages, start, kv_len, q_heads: int, *, max_q=None, max_kv=None,
                    tree_mask=None, blocks=None, rows=None, layer: int = 0, scale=None,
                    out_dtype=BF16, out=None, workspace=None, stream=None):
    """Attention of new tokens over their sequences' pages (nk_attention_paged).

    q bf16 [tokens, q_heads * head_dim]; sequence b's tokens are rows
    start[b] .. start[b+1]-1 and the last ones of its kv_len[b] positions.
    Without masks a token attends every position up to its own; with tree_mask
    (int64 [tokens], bit j: the sequence's new token j) every cached position
    and the drafts of its branch; with blocks (int32 [tokens, kv_heads, n],
    kv_block_select) the listed blocks.  max_q and max_kv bound the new tokens
    and the length of a sequence (defaults: all tokens, but no more than max_kv
    and, with tree_mask, 64; the table's width); close bounds cost less.  Returns
    [tokens, q_heads * head_dim] in bf16, or f32 with out_dtype=F32; rows that
    belong to no sequence stay as they were (a new `out` is not initialised).
    Weights are rounded to bf16 for the product with the values in both.
    workspace: optional uint8 device tensor of attention_paged_workspace_bytes."""
    tokens, ld_q = pages._queries(q, q_heads)
    b = pages.batch(start, kv_len, tokens, max_q, max_kv, rows)
    if max_q is None and tree_mask is not None and b.max_new > 64:
        b.max_new = 64
    return _attend(pages, q, ld_q, b, q_heads, tree_mask, blocks, layer, scale, out_dtype, out,
                   workspace, stream)


def attention_paged_workspace_bytes(pages: KvPages, tokens: int, seqs: int, q_heads: int, *,
                                    max_q: int, max_kv: int, max_blocks: int = 0) -> int:
    """Scratch bytes of attention_paged for these bounds (max_blocks > 0: the
    form with block lists of that width)."""
    return pages._attend_bytes(NkKvBatch(seqs, tokens, 16, 16, 16, max_q, max_kv), q_heads,
                               max_blocks)


def _select(pages, q, ld_q, b, q_heads, top_k, sink, local, layer, out, workspace, stream):
    """kv_block_select behind its checks of q and the batch b."""
    import torch

    dev, tokens = pages.device, q.shape[0]
    if out is None:
        out = _empty((tokens, pages.kv_heads, max(top_k, 1)), torch.int32, dev, stream)
    else:
        _expect(out, "out", torch.int32, 3, dev)
        if out.shape != (tokens, pages.kv_heads, top_k) or not out.is_contiguous():
            raise ValueError("out must be contiguous [tokens, kv_heads, top_k]")
    br = ctypes.byref(b)
    if workspace is None:
        workspace = _empty(pages._select_bytes(b), torch.uint8, dev, stream, result=False)
    _call_on(dev, "nk_kv_block_select", pages._ref, layer, br, q.data_ptr(), ld_q, q_heads, top_k,
             sink, local, out.data_ptr(), workspace.data_ptr(), _bytes_of(workspace, dev),
             _stream_of(dev, stream))
    return out


def kv_block_select(q, pages: KvPages, start, kv_len, q_heads: int, top_k: int, *, sink: int = 1,
                    local: int = 1, max_q=None, max_kv=None, rows=None, layer: int = 0, out=None,
                    workspace=None, stream=None):
    """The blocks each token's query reads (nk_kv_block_select): int32 [tokens,
    kv_heads, top_k], ascending, -1 behind the last; the first `sink` and last
    `local` blocks and those whose key bounds allow the largest scores."""
    tokens, ld_q = pages._queries(q, q_heads)
    b = pages.batch(start, kv_len, tokens, max_q, max_kv, rows)
    return _select(pages, q, ld_q, b, q_heads, top_k, sink, local, layer, out, workspace, stream)


def attention_paged_sparse(q, pages: KvPages, start, kv_len, q_heads: int, top_k: int, *,
                           sink: int = 1, local: int = 1, max_q=None, max_kv=None, rows=None,
                           layer: int = 0, scale=None, out_dtype=BF16, out=None, stream=None):
    """kv_block_select, then attention_paged over the chosen blocks; returns
    (out, blocks)."""
    import torch

    tokens, ld_q = pages._queries(q, q_heads)
    b = pages.batch(start, kv_len, tokens, max_q, max_kv, rows)
    # One workspace for both: the selection is done with it when the attention starts.
    size = max(pages._select_bytes(b), pages._attend_bytes(b, q_heads, top_k))
    workspace = _empty(size, torch.uint8, pages.device, stream, result=False)
    blocks = _select(pages, q, ld_q, b, q_heads, top_k, sink, local, layer, None, workspace,
                     stream)
    return _attend(pages, q, ld_q, b, q_heads, None, blocks, layer, scale, out_dtype, out,
                   workspace, stream), blocks


# ------------------------------------------------- decoder steps around projections
def _dtype_code(t):
    import torch

    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.bfloat16:
        return BF16
    raise TypeError(f"unsupported dtype {t.dtype}")


def embedding_lookup(table, token_ids, vocab_size, hidden_size, *, out=None, out_dtype=None,
                     check=True, stream=None):
    """embedding_lookup (embedding.rs:73-91); token_ids int32 on the device."""
    import torch

    _require_cuda(table, token_ids, out)
    n = token_ids.numel()
    if out is None:
        dt = out_dtype or table.dtype
        out = torch.empty(n, hidden_size, dtype=dt, device=table.device)
    call("nk_embedding_lookup", ptr(table), _dtype_code(table), table.numel(), ptr(token_ids), n,
         vocab_size, hidden_size, ptr(out), _dtype_code(out), out.numel(), 1 if check else 0,
         stream_ptr(stream))
    return out


def add_rms_norm_rows(residual, delta, weight, epsilon, *, h_out=None, normed=None,
                      normed_dtype=BF16, stream=None):
    """Block residual (block.rs:145-151) fused with the next RMSNorm; returns (h, normed)."""
    import torch

    _require_cuda(residual, delta, weight, h_out, normed)
    rows, width = residual.shape
    h_out = residual if h_out is None else h_out
    if normed is None:
        normed = torch.empty(rows, width, device=residual.device,
                             dtype=torch.bfloat16 if normed_dtype == BF16 else torch.float32)
    call("nk_add_rms_norm_rows", ptr(residual), ptr(delta), rows, width, ptr(weight),
         weight.numel(), epsilon, ptr(h_out), ptr(normed), _dtype_code(normed),
         stream_ptr(stream))
    return h_out, normed


def argmax_rows(x, *, out=None, stream=None):
    """predict_next_token's pick (model.rs:325-337) per row of x [rows, n]."""
    import torch

    _require_cuda(x, out)
    rows, n = x.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.int32, device=x.device)
    call("nk_argmax_rows", ptr(x), _dtype_code(x), rows, n, x.stride(0), ptr(out),
         stream_ptr(stream))
    return out
