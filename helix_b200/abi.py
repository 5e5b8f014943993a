"""ctypes mirror of include/helix/helix.h.

Field order, types and enum values follow the C header exactly; the header in
turn keeps the reference ABI (reference include/helix/helix.h:42-218).
``load()`` opens the in-tree ``libhelix.so`` and raises when it is missing: the
package has no fallback implementation.
"""
from __future__ import annotations

import ctypes as C
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libhelix.so"

# helix_status
HELIX_OK = 0
HELIX_ERR_UNSUPPORTED_SHAPE = 1
HELIX_ERR_NO_DEVICE = 2
HELIX_ERR_SCRATCH_TOO_SMALL = 3
HELIX_ERR_INVALID_ARG = 4
HELIX_ERR_PIPELINE = 5
STATUS_NAMES = {0: "OK", 1: "UNSUPPORTED_SHAPE", 2: "NO_DEVICE", 3: "SCRATCH_TOO_SMALL",
                4: "INVALID_ARG", 5: "PIPELINE"}

# helix_dtype
HELIX_F32, HELIX_F16, HELIX_BF16, HELIX_E4M3 = 0, 1, 2, 3
# helix_a_form
HELIX_A_SCALAR_PER_HEAD, HELIX_A_DIAG_PER_CHANNEL = 0, 1
# helix_backend
HELIX_BACKEND_AUTO, HELIX_BACKEND_SGMMA, HELIX_BACKEND_MPP, HELIX_BACKEND_REF = 0, 1, 2, 3
# include/helix/helix_block.h: values that share a scale; helix_scale_form
HELIX_GROUP = 128
HELIX_SCALE_ROWS, HELIX_SCALE_BLOCKS = 0, 1
HELIX_GATED_CHUNK = 128

I32, I64 = C.c_int32, C.c_int64


class ScanDesc(C.Structure):
    """helix_scan_desc."""
    _fields_ = [
        ("n_tok", I32), ("n_seq", I32), ("n_head", I32), ("head_dim", I32),
        ("d_state", I32), ("n_group", I32),
        ("s_x", I64 * 3), ("s_b", I64 * 3), ("s_c", I64 * 3), ("s_dt", I64 * 2),
        ("s_s", I64 * 3), ("s_y", I64 * 3), ("s_a", I64),
        ("seq_x", I64), ("seq_b", I64), ("seq_c", I64), ("seq_dt", I64),
        ("seq_s", I64), ("seq_y", I64),
        ("chunk", I32), ("a_form", C.c_int), ("io_dtype", C.c_int),
        ("compute_dtype", C.c_int), ("backend", C.c_int), ("multipass", C.c_bool),
        ("dt_min", C.c_float), ("dt_max", C.c_float),
    ]

    def copy(self) -> "ScanDesc":
        d = ScanDesc()
        C.memmove(C.byref(d), C.byref(self), C.sizeof(ScanDesc))
        return d


class Tensor(C.Structure):
    """helix_tensor: device pointer + byte offset."""
    _fields_ = [("buf", C.c_void_p), ("offset", C.c_uint64)]


NULL_TENSOR = Tensor(None, 0)

# Every entry point include/helix/*.h declares.
EXPORTS = (
    "helix_scan_desc_init", "helix_ctx_create", "helix_ctx_free", "helix_ctx_last_error",
    "helix_ctx_select_backend", "helix_ctx_backend_desc", "helix_scan_supported",
    "helix_scan_scratch_size", "helix_scan_encode", "helix_scan_encode_into",
    # include/helix/helix_ext.h
    "helix_device_fault", "helix_scan_encode_static",
    "helix_scan_shard_state_scratch_size", "helix_scan_shard_state", "helix_scan_carry_combine",
    "helix_scan_plan_info", "helix_scan_encode_shard",
    # include/helix/helix_block.h
    "helix_rms_norm_desc_init", "helix_rms_norm_encode", "helix_rms_norm_grad_scratch_size",
    "helix_rms_norm_grad_encode", "helix_quant8_desc_init", "helix_quant8_encode",
    "helix_matmul8_desc_init", "helix_matmul8_encode",
    "helix_gated_scan_desc_init", "helix_gated_scan_states_size", "helix_gated_scan_encode",
    "helix_gated_scan_grad_encode",
)


class RmsNormDesc(C.Structure):
    """helix_rms_norm_desc (include/helix/helix_block.h)."""
    _fields_ = [("n_row", I64), ("n_col", I32), ("eps", C.c_float), ("x_dtype", C.c_int), ("sum_dtype", C.c_int),
                ("out_dtype", C.c_int), ("w_dtype", C.c_int), ("ld_x", I64), ("ld_res", I64), ("ld_sum", I64),
                ("ld_out", I64), ("ld_scale", I64), ("ld_dout", I64), ("ld_dsum", I64), ("ld_dx", I64),
                ("ld_dres", I64)]


class Quant8Desc(C.Structure):
    """helix_quant8_desc (include/helix/helix_block.h)."""
    _fields_ = [("n_row", I64), ("n_col", I64), ("x_dtype", C.c_int), ("form", C.c_int), ("transpose", C.c_bool),
                ("ld_x", I64), ("ld_q", I64), ("ld_scale", I64)]


class Matmul8Desc(C.Structure):
    """helix_matmul8_desc (include/helix/helix_block.h)."""
    _fields_ = [("m", I32), ("n", I32), ("k", I32), ("b_form", C.c_int), ("out_dtype", C.c_int), ("ld_a", I64),
                ("ld_b", I64), ("ld_out", I64), ("ld_a_scale", I64), ("ld_b_scale", I64)]


class GatedScanDesc(C.Structure):
    """helix_gated_scan_desc (include/helix/helix_block.h)."""
    _fields_ = [("n_tok", I32), ("n_seq", I32), ("n_chan", I32), ("io_dtype", C.c_int)] + [
        (n, I64) for n in ("s_v", "s_g", "s_y", "s_dy", "s_dv", "s_dg", "seq_v", "seq_g", "seq_y", "seq_dy",
                           "seq_dv", "seq_dg", "seq_h0", "seq_h1", "seq_dh1", "seq_dh0")]


class PlanInfo(C.Structure):
    """helix_plan_info (include/helix/helix_ext.h)."""
    _fields_ = [("family", I32), ("chunk", I32), ("run_tokens", I32), ("n_runs", I32),
                ("runs_per_span", I32), ("n_spans", I32), ("state_runs", I32), ("reserved", I32),
                ("scratch_bytes", C.c_uint64)]

_lib = None


def load(path: Path | str | None = None) -> C.CDLL:
    """Opens libhelix.so and declares prototypes.  Raises if it is absent."""
    global _lib
    if _lib is not None and path is None:
        return _lib
    p = Path(path) if path else LIB_PATH
    if not p.exists():
        raise RuntimeError(f"{p} is missing: build it with `python -m helix_b200.build`")
    lib = C.CDLL(str(p))
    P = C.POINTER
    lib.helix_scan_desc_init.argtypes = [P(ScanDesc), I32, I32, I32, I32, I32, I32]
    lib.helix_scan_desc_init.restype = None
    lib.helix_ctx_create.argtypes = [P(C.c_void_p), C.c_void_p, C.c_char_p]
    lib.helix_ctx_create.restype = C.c_int
    lib.helix_ctx_free.argtypes = [C.c_void_p]
    lib.helix_ctx_free.restype = None
    lib.helix_ctx_last_error.argtypes = [C.c_void_p]
    lib.helix_ctx_last_error.restype = C.c_char_p
    lib.helix_ctx_select_backend.argtypes = [C.c_void_p, P(ScanDesc)]
    lib.helix_ctx_select_backend.restype = C.c_int
    lib.helix_ctx_backend_desc.argtypes = [C.c_void_p, P(ScanDesc)]
    lib.helix_ctx_backend_desc.restype = C.c_char_p
    lib.helix_scan_supported.argtypes = [C.c_void_p, P(ScanDesc)]
    lib.helix_scan_supported.restype = C.c_bool
    lib.helix_scan_scratch_size.argtypes = [C.c_void_p, P(ScanDesc)]
    lib.helix_scan_scratch_size.restype = C.c_size_t
    enc = [C.c_void_p, C.c_void_p, P(ScanDesc)] + [Tensor] * 10
    lib.helix_scan_encode.argtypes = enc
    lib.helix_scan_encode.restype = C.c_int
    lib.helix_scan_encode_into.argtypes = enc
    lib.helix_scan_encode_into.restype = C.c_int
    lib.helix_device_fault.argtypes = [C.c_void_p, P(C.c_uint32)]
    lib.helix_device_fault.restype = C.c_int
    lib.helix_scan_encode_static.argtypes = [C.c_void_p, C.c_void_p, P(ScanDesc)] + [Tensor] * 9
    lib.helix_scan_encode_static.restype = C.c_int
    lib.helix_scan_shard_state_scratch_size.argtypes = [C.c_void_p, P(ScanDesc)]
    lib.helix_scan_shard_state_scratch_size.restype = C.c_size_t
    lib.helix_scan_shard_state.argtypes = [C.c_void_p, C.c_void_p, P(ScanDesc)] + [Tensor] * 8
    lib.helix_scan_shard_state.restype = C.c_int
    lib.helix_scan_carry_combine.argtypes = [C.c_void_p, C.c_void_p, P(ScanDesc)] + [Tensor] * 4 + [
        C.c_uint32, Tensor]
    lib.helix_scan_carry_combine.restype = C.c_int
    lib.helix_scan_encode_shard.argtypes = [C.c_void_p, C.c_void_p, P(ScanDesc)] + [Tensor] * 9
    lib.helix_scan_encode_shard.restype = C.c_int
    lib.helix_scan_plan_info.argtypes = [C.c_void_p, P(ScanDesc), P(PlanInfo)]
    lib.helix_scan_plan_info.restype = C.c_int
    lib.helix_rms_norm_desc_init.argtypes = [P(RmsNormDesc), I64, I32]
    lib.helix_rms_norm_desc_init.restype = None
    lib.helix_rms_norm_encode.argtypes = [C.c_void_p, C.c_void_p, P(RmsNormDesc)] + [Tensor] * 7
    lib.helix_rms_norm_encode.restype = C.c_int
    lib.helix_rms_norm_grad_scratch_size.argtypes = [C.c_void_p, P(RmsNormDesc)]
    lib.helix_rms_norm_grad_scratch_size.restype = C.c_size_t
    lib.helix_rms_norm_grad_encode.argtypes = [C.c_void_p, C.c_void_p, P(RmsNormDesc)] + [Tensor] * 9
    lib.helix_rms_norm_grad_encode.restype = C.c_int
    lib.helix_quant8_desc_init.argtypes = [P(Quant8Desc), I64, I64, C.c_int, C.c_bool]
    lib.helix_quant8_desc_init.restype = None
    lib.helix_quant8_encode.argtypes = [C.c_void_p, C.c_void_p, P(Quant8Desc)] + [Tensor] * 3
    lib.helix_quant8_encode.restype = C.c_int
    lib.helix_matmul8_desc_init.argtypes = [P(Matmul8Desc), I32, I32, I32, C.c_int]
    lib.helix_matmul8_desc_init.restype = None
    lib.helix_matmul8_encode.argtypes = [C.c_void_p, C.c_void_p, P(Matmul8Desc)] + [Tensor] * 5
    lib.helix_matmul8_encode.restype = C.c_int
    lib.helix_gated_scan_desc_init.argtypes = [P(GatedScanDesc), I32, I32, I32]
    lib.helix_gated_scan_desc_init.restype = None
    lib.helix_gated_scan_states_size.argtypes = [P(GatedScanDesc)]
    lib.helix_gated_scan_states_size.restype = C.c_size_t
    lib.helix_gated_scan_encode.argtypes = [C.c_void_p, C.c_void_p, P(GatedScanDesc)] + [Tensor] * 7
    lib.helix_gated_scan_encode.restype = C.c_int
    lib.helix_gated_scan_grad_encode.argtypes = [C.c_void_p, C.c_void_p, P(GatedScanDesc)] + [Tensor] * 9
    lib.helix_gated_scan_grad_encode.restype = C.c_int
    if path is None:
        _lib = lib
    return lib


def desc_init(L: int, S: int, H: int, P: int, N: int, G: int) -> ScanDesc:
    d = ScanDesc()
    load().helix_scan_desc_init(C.byref(d), L, S, H, P, N, G)
    return d
