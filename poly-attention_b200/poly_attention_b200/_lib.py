"""ctypes binding of libpolyattn.so (declarations: include/poly_attention.h).

The library is the only implementation: if it is missing, importing this
module raises, there is no fallback.
"""
from __future__ import annotations

import ctypes
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libpolyattn.so")

POLY_OK, POLY_EINVAL, POLY_EUNSUPPORTED, POLY_ECUDA = 0, 1, 2, 3
POLY_F32, POLY_F16, POLY_BF16 = 0, 1, 2
ABI_VERSION = 2

c_i32, c_i64, c_f32, c_vp, c_sz = ctypes.c_int32, ctypes.c_int64, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t
I64x3 = c_i64 * 3
I64x2 = c_i64 * 2


class PolyPassArgs(ctypes.Structure):
    _fields_ = [
        ("batch", c_i32), ("heads", c_i32), ("kv_heads", c_i32), ("seq_q", c_i32), ("seq_k", c_i32),
        ("head_dim", c_i32), ("dtype", c_i32), ("causal", c_i32), ("scale", c_f32), ("softclamp", c_f32),
        ("q", c_vp), ("q_stride", I64x3),
        ("k", c_vp), ("k_stride", I64x3),
        ("v", c_vp), ("v_stride", I64x3),
        ("v_mul", c_vp), ("v_mul_stride", I64x3),
        ("bias", c_vp), ("bias_stride", I64x2),
        ("key_mask", c_vp), ("key_mask_stride", c_i64),
        ("query_mask", c_vp), ("query_mask_stride", c_i64),
        ("out", c_vp), ("out_stride", I64x3),
        ("lse", c_vp), ("lse_stride", I64x2),
        ("epi_mul", c_vp), ("epi_mul_stride", I64x3),
        ("epi_out", c_vp), ("epi_out_stride", I64x3),
        ("workspace", c_vp), ("workspace_bytes", c_sz),
        ("causal_offset", c_i32), ("reserved_", c_i32),
    ]


class PolyPassBwdArgs(ctypes.Structure):
    _fields_ = [
        ("fwd", PolyPassArgs),
        ("dout", c_vp), ("dout_stride", I64x3),
        ("dlse", c_vp), ("dlse_stride", I64x2),
        ("dq", c_vp), ("dq_stride", I64x3),
        ("dk", c_vp), ("dk_stride", I64x3),
        ("dv", c_vp), ("dv_stride", I64x3),
        ("dbias", c_vp), ("dbias_stride", I64x2),
        ("dq_accumulate", c_i32), ("reserved", c_i32),
        ("workspace", c_vp), ("workspace_bytes", c_sz),
    ]


class PolyMergeArgs(ctypes.Structure):
    _fields_ = [
        ("parts", c_i32), ("head_dim", c_i32), ("dtype", c_i32), ("reserved", c_i32), ("rows", c_i64),
        ("part_out", c_vp), ("part_lse", c_vp), ("out", c_vp), ("lse", c_vp),
    ]


class PolyRowCopy(ctypes.Structure):
    _fields_ = [("src", c_vp), ("dst", c_vp), ("outer", ctypes.c_int32), ("inner", ctypes.c_int32),
                ("row_bytes", ctypes.c_int32), ("reserved", ctypes.c_int32),
                ("src_stride", ctypes.c_int64 * 2), ("dst_stride", ctypes.c_int64 * 2)]


MAX_ROW_COPIES = 16


class PolyHeadNorm(ctypes.Structure):
    _fields_ = [("src", c_vp), ("dst", c_vp), ("weight", c_vp), ("batch", ctypes.c_int32),
                ("heads", ctypes.c_int32), ("rows", ctypes.c_int32), ("dim", ctypes.c_int32),
                ("src_stride", ctypes.c_int64 * 3), ("src_dtype", ctypes.c_int32), ("dst_dtype", ctypes.c_int32),
                ("weight_dtype", ctypes.c_int32), ("eps", ctypes.c_float)]


MAX_NORMS = 4


class PolyPackedArgs(ctypes.Structure):
    _fields_ = [("fwd", PolyPassArgs), ("cu_seqlens", c_vp), ("seqs", c_i32), ("max_len", c_i32),
                ("zero_rest", c_i32), ("reserved", c_i32), ("out_lo", c_vp)]


class PolyPackedBwdArgs(ctypes.Structure):
    _fields_ = [("bwd", PolyPassBwdArgs), ("cu_seqlens", c_vp), ("seqs", c_i32), ("max_len", c_i32),
                ("zero_rest", c_i32), ("reserved", c_i32), ("out_lo", c_vp),
                ("v_left", c_vp), ("v_left_stride", I64x2), ("v_right", c_vp), ("v_right_stride", I64x2),
                ("dv_right", c_vp), ("dv_right_stride", I64x2)]


MAX_TREE_NODES = 64
MAX_TREE_CACHES = 16


class PolyTreePass(ctypes.Structure):
    _fields_ = [
        ("batch", c_i32), ("heads", c_i32), ("kv_heads", c_i32), ("nodes", c_i32), ("head_dim", c_i32), ("dtype", c_i32),
        ("capacity", c_i32), ("reserved", c_i32), ("scale", c_f32), ("softclamp", c_f32),
        ("q", c_vp), ("q_stride", I64x3), ("k", c_vp), ("k_stride", I64x3), ("v", c_vp), ("v_stride", I64x3),
        ("v_mul", c_vp), ("v_mul_stride", I64x3), ("bias", c_vp), ("bias_stride", I64x2),
        ("lengths", c_vp), ("parents", c_vp), ("parents_stride", c_i64),
        ("out", c_vp), ("out_stride", I64x3), ("lse", c_vp), ("lse_stride", I64x2),
        ("cache_out", c_vp), ("cache_out_stride", I64x3), ("cache_lse", c_vp), ("cache_lse_stride", I64x2),
        ("workspace", c_vp), ("workspace_bytes", c_sz),
    ]


class _TreeAppendRow(ctypes.Structure):
    _fields_ = [("src", c_vp), ("src_stride", I64x3), ("cache", c_vp), ("cache_stride", I64x3)]


class PolyTreeAppend(ctypes.Structure):
    _fields_ = [("batch", c_i32), ("kv_heads", c_i32), ("nodes", c_i32), ("row_bytes", c_i32), ("capacity", c_i32),
                ("n", c_i32), ("lengths", c_vp), ("parents", c_vp), ("parents_stride", c_i64),
                ("t", _TreeAppendRow * MAX_TREE_CACHES)]


class _TreeCommitRow(ctypes.Structure):
    _fields_ = [("cache", c_vp), ("cache_stride", I64x3), ("row_bytes", c_i64)]


class PolyTreeCommit(ctypes.Structure):
    _fields_ = [("batch", c_i32), ("kv_heads", c_i32), ("nodes", c_i32), ("capacity", c_i32), ("n", c_i32),
                ("path_len", c_i32), ("lengths", c_vp), ("path", c_vp), ("path_stride", c_i64), ("count", c_vp),
                ("t", _TreeCommitRow * MAX_TREE_CACHES)]


class PolyRotaryTensor(ctypes.Structure):
    _fields_ = [("src", c_vp), ("dst", c_vp), ("heads", c_i32), ("reserved", c_i32),
                ("src_stride", I64x3), ("dst_stride", I64x3)]


MAX_ROTARY = 8


class PolyRotaryArgs(ctypes.Structure):
    _fields_ = [
        ("batch", c_i32), ("rows", c_i32), ("dim", c_i32), ("rot", c_i32), ("dtype", c_i32), ("interleaved", c_i32),
        ("inverse", c_i32), ("n", c_i32), ("factor", c_f32), ("pos_wide", c_i32),
        ("positions", c_vp), ("pos_stride", I64x2), ("pos_start", c_i64),
        ("inv_freq", c_vp), ("angles", c_vp), ("angle_stride", I64x2),
        ("cu_seqlens", c_vp), ("seqs", c_i32), ("reserved", c_i32),
        ("t", PolyRotaryTensor * MAX_ROTARY),
    ]


def packer(cls, before=None):
    """struct.Struct of a ctypes Structure (of its fields before ``before``, if given) without nested arrays of
    structures: argument blocks of calls whose latency counts are packed in one go (some 60 attribute writes
    cost more than the launch)."""
    codes = {c_i32: "i", c_i64: "q", c_f32: "f", c_vp: "Q", c_sz: "Q"}

    def flat(t):
        if issubclass(t, ctypes.Structure):
            return "".join(flat(f[1]) for f in t._fields_)
        if issubclass(t, ctypes.Array):
            return flat(t._type_) * t._length_
        return codes[t]
    names = [f[0] for f in cls._fields_]
    fields = cls._fields_[:names.index(before)] if before else cls._fields_
    st = struct.Struct("@" + "".join(flat(f[1]) for f in fields))
    if st.size > (getattr(cls, before).offset if before else ctypes.sizeof(cls)):
        raise ImportError(f"cannot pack {cls.__name__}")
    return st


EXPORTS = {
    "poly_pass_fwd": (ctypes.c_int, [ctypes.POINTER(PolyPassArgs), c_vp]),
    "poly_pass_fwd_workspace_size": (c_sz, [ctypes.POINTER(PolyPassArgs)]),
    "poly_pass_bwd": (ctypes.c_int, [ctypes.POINTER(PolyPassBwdArgs), c_vp]),
    "poly_pass_bwd_workspace_size": (c_sz, [ctypes.POINTER(PolyPassBwdArgs)]),
    "poly_lse_merge": (ctypes.c_int, [ctypes.POINTER(PolyMergeArgs), c_vp]),
    "poly_decode_chain": (ctypes.c_int, [ctypes.POINTER(PolyPassArgs), ctypes.c_int, c_vp]),
    "poly_copy_rows": (ctypes.c_int, [ctypes.POINTER(PolyRowCopy), ctypes.c_int, c_vp]),
    "poly_head_rmsnorm": (ctypes.c_int, [ctypes.POINTER(PolyHeadNorm), ctypes.c_int, c_vp]),
    "poly_packed_pass_fwd": (ctypes.c_int, [ctypes.POINTER(PolyPackedArgs), c_vp]),
    "poly_packed_pass_bwd": (ctypes.c_int, [ctypes.POINTER(PolyPackedBwdArgs), c_vp]),
    "poly_packed_pass_bwd_workspace_size": (c_sz, [ctypes.POINTER(PolyPackedBwdArgs)]),
    "poly_packed_pass_fwd_kernel_name": (ctypes.c_char_p, [ctypes.POINTER(PolyPackedArgs)]),
    "poly_packed_pass_bwd_kernel_name": (ctypes.c_char_p, [ctypes.POINTER(PolyPackedBwdArgs)]),
    "poly_tree_chain": (ctypes.c_int, [ctypes.POINTER(PolyTreeAppend), ctypes.POINTER(PolyTreePass), ctypes.c_int, c_vp]),
    "poly_tree_chain_counted": (ctypes.c_int, [ctypes.POINTER(PolyTreeAppend), ctypes.POINTER(PolyTreePass), ctypes.c_int, c_vp,
                                               c_vp]),
    "poly_tree_workspace_size": (c_sz, [ctypes.POINTER(PolyTreePass)]),
    "poly_tree_commit": (ctypes.c_int, [ctypes.POINTER(PolyTreeCommit), c_vp]),
    "poly_tree_commit_counted": (ctypes.c_int, [ctypes.POINTER(PolyTreeCommit), c_vp, c_vp]),
    "poly_tree_positions": (ctypes.c_int, [c_vp, c_vp, c_i64, c_i32, c_i32, c_vp, c_i64, c_vp]),
    "poly_tree_kernel_name": (ctypes.c_char_p, [ctypes.POINTER(PolyTreePass)]),
    "poly_rotary": (ctypes.c_int, [ctypes.POINTER(PolyRotaryArgs), c_vp]),
    "poly_pass_bwd_noalloc": (ctypes.c_int, [ctypes.POINTER(PolyPassBwdArgs), c_vp]),
    "poly_noalloc_scratch_bytes": (c_sz, []),
    "poly_pass_fwd_kernel_name": (ctypes.c_char_p, [ctypes.POINTER(PolyPassArgs)]),
    "poly_pass_bwd_kernel_name": (ctypes.c_char_p, [ctypes.POINTER(PolyPassBwdArgs)]),
    "poly_last_error": (ctypes.c_char_p, []),
    "poly_launch_count": (ctypes.c_ulonglong, []),
    "poly_device_error": (ctypes.c_int, [ctypes.POINTER(ctypes.c_int), ctypes.c_int]),
    "poly_selftest_wait_timeout": (ctypes.c_int, [ctypes.c_ulonglong, c_vp, c_vp]),
    "poly_abi_version": (ctypes.c_int, []),
    "poly_sizeof_pass_args": (c_sz, []),
    "poly_sizeof_pass_bwd_args": (c_sz, []),
    "poly_sizeof_merge_args": (c_sz, []),
    "poly_sizeof_rotary_args": (c_sz, []),
    "poly_sizeof_packed_args": (c_sz, []),
    "poly_sizeof_packed_bwd_args": (c_sz, []),
    "poly_sizeof_tree_pass": (c_sz, []),
    "poly_sizeof_tree_append": (c_sz, []),
    "poly_sizeof_tree_commit": (c_sz, []),
}


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError(f"{LIB_PATH} is missing: build it with `python poly-attention_b200/build.py` "
                          "(there is no non-CUDA implementation)")
    lib = ctypes.CDLL(LIB_PATH)
    for name, (res, args) in EXPORTS.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    if lib.poly_abi_version() != ABI_VERSION:
        raise ImportError("libpolyattn.so ABI version mismatch")
    for fn, st in (("poly_sizeof_pass_args", PolyPassArgs), ("poly_sizeof_pass_bwd_args", PolyPassBwdArgs),
                   ("poly_sizeof_merge_args", PolyMergeArgs), ("poly_sizeof_rotary_args", PolyRotaryArgs),
                   ("poly_sizeof_packed_args", PolyPackedArgs), ("poly_sizeof_packed_bwd_args", PolyPackedBwdArgs),
                   ("poly_sizeof_tree_pass", PolyTreePass), ("poly_sizeof_tree_append", PolyTreeAppend),
                   ("poly_sizeof_tree_commit", PolyTreeCommit)):
        if getattr(lib, fn)() != ctypes.sizeof(st):
            raise ImportError(f"libpolyattn.so struct layout mismatch ({st.__name__})")
    return lib


lib = _load()


def check(rc: int, what: str):
    if rc == POLY_OK:
        return
    msg = f"{what}: {lib.poly_last_error().decode()}"
    if rc == POLY_EINVAL:
        raise ValueError(msg)
    if rc == POLY_EUNSUPPORTED:
        raise NotImplementedError(msg)
    raise RuntimeError(msg)


def launch_count() -> int:
    """Kernels launched by libpolyattn.so in this process so far."""
    return int(lib.poly_launch_count())


def device_error(reset: bool = False) -> int:
    """Device error word (non-zero: a bounded in-kernel wait gave up)."""
    v = ctypes.c_int(0)
    check(lib.poly_device_error(ctypes.byref(v), int(reset)), "poly_device_error")
    return v.value
