"""exl3c4.py -- Python binding of libexl3c4.so (include/exl3c4.h) for tests and the benchmark.

The library is C over HIP; this module only marshals pointers. torch is used for device memory and the stream
(plumbing), never for the computation: every op runs in the library's HIP kernels. If libexl3c4.so is missing this
module raises -- there is no fallback of any kind.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libexl3c4.so")

DOWN, GATE_UP, PREP_GU, GU_DN = 0, 1, 2, 3
K_PREP, K_GATE_UP, K_EPI_GU, K_DOWN, K_GATE_UP_DOWN = 0, 1, 2, 3, 4
GD_FUSE_MIN_T = 32                  # gate_up_down runs as one kernel at decode from this many sorted rows
CB = {"3inst": 0, "mcg": 1, "mul1": 2}
F16, BF16 = 0, 1
MX4 = 3
ACT_NONE, ACT_SWIGLU = 0, 1
STATUS = {0: "OK", -1: "RAD_E_SHAPE", -2: "RAD_E_DTYPE", -3: "RAD_E_ALIGN", -4: "RAD_E_STRIDE", -9: "RAD_E_SCHEMA",
          -12: "RAD_E_INVAL", -18: "RAD_E_UNSUPPORTED", -20: "RAD_E_SCRATCH", -21: "RAD_E_DEVICE",
          -5: "RAD_E_FORMAT", -30: "RAD_E_NOTFOUND", -31: "RAD_E_IO"}
E_FORMAT, E_NOTFOUND, E_IO = -5, -30, -31

_lib = None
_p = C.c_void_p
_i64 = C.c_int64
_i32 = C.c_int32


class Class(C.Structure):
    _fields_ = [("rows", _i32), ("cols", _i32),
                ("codes", _p), ("suh", _p), ("suh1", _p), ("svh", _p), ("dn_suh", _p),
                ("codes_stride", _i64), ("suh_stride", _i64), ("suh1_stride", _i64), ("svh_stride", _i64),
                ("dn_suh_stride", _i64)]


class Op(C.Structure):
    _fields_ = [("op", _i32), ("bits", _i32), ("codebook", _i32), ("n_class", _i32), ("h_rot", _i32), ("a_rot", _i32),
                ("M", _i64), ("n_expert", _i64), ("top_k", _i64),
                ("cls", Class * 4), ("dn", Class * 4),
                ("x", _p), ("x_dtype", _i32), ("x_rows", _i64), ("x_cols", _i64), ("x_pitch", _i64),
                ("sorted_tok", _p), ("expert_offset", _p),
                ("y", _p), ("T", _i64), ("y_cols", _i64), ("y_pitch", _i64), ("dn_bits", _i32)]


class Gemm(C.Structure):
    _fields_ = [("x_type", _i32), ("w_type", _i32), ("y_type", _i32), ("act", _i32),
                ("N", _i64), ("K", _i64), ("n_expert", _i64), ("top_k", _i64), ("T", _i64),
                ("x", _p), ("x_scales", _p), ("x_rows", _i64), ("x_pitch", _i64), ("xs_pitch", _i64),
                ("w", _p), ("w_scales", _p), ("w_pitch", _i64), ("ws_pitch", _i64), ("w_stride", _i64),
                ("ws_stride", _i64), ("sorted_tok", _p), ("expert_offset", _p), ("y", _p), ("y_pitch", _i64)]


class Mx4:
    """MX4 rows (include/exl3c4.h) of values [..., rows, cols]: codes uint8 [..., rows, >= 16 ceil(cols / 32)], scales uint8
    [..., rows, >= ceil(cols / 32)], the columns they stand for. Its attributes are fixed, and the planes keep their sizes and
    strides (the conversions take a row's pitches from them once); where their memory is, is read at each call. Leading
    dimensions have to step evenly as one for the conversions (for moe_gemm they need not)."""
    __slots__ = ("codes", "scales", "cols", "shape", "rows", "device", "_pitches")

    def __init__(self, codes, scales, cols: int):
        nb = (cols + 31) // 32
        if codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] < 16 * nb or scales.shape[-1] < nb or \
                codes.element_size() != 1 or scales.element_size() != 1 or codes.device != scales.device:
            raise ValueError("the MX4 planes do not fit each other or their columns")
        put = super().__setattr__
        put("codes", codes)
        put("scales", scales)
        put("cols", cols)
        put("shape", codes.shape[:-1] + (cols,))
        put("rows", codes.shape[:-1].numel())
        put("device", codes.get_device())
        put("_pitches", None)

    def __setattr__(self, name, *value):
        raise AttributeError(f"{name} of an Mx4 is fixed: make another one")

    __delattr__ = __setattr__

    def __reduce__(self):                                      # copies and pickles: made of their own planes
        return Mx4, (self.codes, self.scales, self.cols)

    def pitches(self):
        if self._pitches is None:
            super().__setattr__("_pitches", (_rows(self.codes)[1], _rows(self.scales)[1]))
        return self._pitches


def lib():
    """The loaded library; raises when it has not been built (no CPU or torch fallback exists)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is not built: run `python -c 'import __graft_entry__ as g; g.build()'`")
        L = C.CDLL(LIB_PATH)
        L.exl3c4_scratch_bytes.restype = _i64
        L.exl3c4_scratch_bytes.argtypes = [C.POINTER(Op)]
        L.exl3c4_launch_scratch_bytes.restype = _i64
        L.exl3c4_launch_scratch_bytes.argtypes = [C.POINTER(Op)]
        L.exl3c4_scratch_bytes_geom.restype = _i64
        L.exl3c4_scratch_bytes_geom.argtypes = [_i32, _i32, C.POINTER(_i32), C.POINTER(_i32), _i64, _i64, _i64]
        L.exl3c4_launch.restype = C.c_int
        L.exl3c4_launch.argtypes = [C.POINTER(Op), _p, _i64, _p]
        L.exl3c4_launch_noalloc.restype = C.c_int
        L.exl3c4_launch_noalloc.argtypes = [C.POINTER(Op), _p]
        L.exl3c4_noalloc_scratch_bytes.restype = _i64
        L.exl3c4_noalloc_scratch_bytes.argtypes = []
        L.exl3c4_launch_checked.restype = C.c_int
        L.exl3c4_launch_checked.argtypes = [C.POINTER(Op), _p, _i64, _p]
        L.exl3c4_dequant.restype = C.c_int
        L.exl3c4_dequant.argtypes = [_p, _i32, _i32, _i32, _i32, _p, _i64, _p]
        L.exl3c4_record_bytes.restype = _i64
        L.exl3c4_record_bytes.argtypes = [_i64, _i64, _i32]
        L.exl3c4_relayout.restype = C.c_int
        L.exl3c4_relayout.argtypes = [_p, _i64, _i64, _i64, _i32, _p]
        L.exl3c4_unrelayout.restype = C.c_int
        L.exl3c4_unrelayout.argtypes = [_p, _i64, _i64, _i32, _p, _i64]
        L.exl3c4_launch_timed.restype = C.c_int
        L.exl3c4_launch_timed.argtypes = [C.POINTER(Op), _p, _i64, _p, _i32, _p, _p]
        L.exl3c4_scratch_partials.restype = C.c_int
        L.exl3c4_scratch_partials.argtypes = [C.POINTER(Op), _i32, C.POINTER(_i64), C.POINTER(_i64), C.POINTER(_i64),
                                              C.POINTER(_i32)]
        L.exl3c4_router_topk.restype = C.c_int
        L.exl3c4_router_topk.argtypes = [_p, _i32, _i64, _i64, _i64, _i32, _i32, _p, _p, _p]
        L.exl3c4_moe_scatter.restype = C.c_int
        L.exl3c4_moe_scatter.argtypes = [_p, _i64, _i32, _i64, _i64, _p, _p, _p, _p, _p]
        L.exl3c4_router_topk_scatter.restype = C.c_int
        L.exl3c4_router_topk_scatter.argtypes = [_p, _i32, _i64, _i64, _i64, _i32, _i32, _p, _p, _p, _p, _p, _p, _p]
        L.exl3c4_moe_gather.restype = C.c_int
        L.exl3c4_moe_gather.argtypes = [_p, _i32, _i64, _p, _p, _i64, _i32, _i64, _p, _i64, _p]
        L.exl3c4_ctr_bytes.restype = _i64
        L.exl3c4_ctr_bytes.argtypes = [C.POINTER(Op)]
        L.exl3c4_launch_ctr.restype = C.c_int
        L.exl3c4_launch_ctr.argtypes = [C.POINTER(Op), _p, _i64, _p, _p, _i64]
        L.exl3c4_launch_gather.restype = C.c_int
        L.exl3c4_launch_gather.argtypes = [C.POINTER(Op), _p, _i64, _p, _p, _i64, _p, _p, _p, _i64]
        L.exl3c4_launch_leaving.restype = C.c_int
        L.exl3c4_launch_leaving.argtypes = [C.POINTER(Op), _p, _i64, _p, _p, _i64, _p, _p, _p, _i64, _i32]
        L.exl3c4_scratch_status.restype = C.c_int
        L.exl3c4_scratch_status.argtypes = [C.POINTER(Op), C.POINTER(_i64)]
        L.exl3c4_record_to_codes.restype = C.c_int
        L.exl3c4_record_to_codes.argtypes = [_p, _i64, _i64, _i32, _p, _i64]
        L.exl3c4_ckpt_open.restype = C.c_int
        L.exl3c4_ckpt_open.argtypes = [C.c_char_p, C.POINTER(_p)]
        L.exl3c4_ckpt_close.restype = None
        L.exl3c4_ckpt_close.argtypes = [_p]
        L.exl3c4_ckpt_layers.restype = _i64
        L.exl3c4_ckpt_layers.argtypes = [_p]
        L.exl3c4_import_parse_name.restype = C.c_int
        L.exl3c4_import_parse_name.argtypes = [C.c_char_p, C.POINTER(_i32), C.POINTER(_i64), C.POINTER(_i32)]
        L.exl3c4_import_weight.restype = C.c_int
        L.exl3c4_import_weight.argtypes = [_p, C.c_char_p, _i32, _i32, _i64, _i64, _p, _i64, _p, _p, _p]
        L.exl3c4_prefill_min_rows.restype = _i64
        L.exl3c4_prefill_min_rows.argtypes = [_i64]
        L.exl3c4_check_narrow.restype = C.c_int
        L.exl3c4_check_narrow.argtypes = [_p, _p, _p, _i64, _p]
        L.exl3c4_mx4_quant.restype = C.c_int
        L.exl3c4_mx4_quant.argtypes = [_p, _i32, _i64, _i64, _i64, _p, _i64, _p, _i64, _p]
        L.exl3c4_mx4_dequant.restype = C.c_int
        L.exl3c4_mx4_dequant.argtypes = [_p, _i64, _p, _i64, _i64, _i64, _p, _i32, _i64, _p]
        L.exl3c4_moe_gemm.restype = C.c_int
        L.exl3c4_moe_gemm.argtypes = [C.POINTER(Gemm), _p]
        L.exl3c4_build_target.restype = C.c_char_p
        L.exl3c4_abi_version.restype = C.c_int
        _lib = L
    return _lib


# ------------------------------------------------------------------------------------------ stored form (host)
def relayout(codes: np.ndarray, rows: int, cols: int, bits: int) -> np.ndarray:
    """Canonical uK plane [rows][row_bytes] -> the stored record (uint8 [rows*cols*bits/8])."""
    codes = np.ascontiguousarray(codes, dtype=np.uint8)
    out = np.zeros(rows * cols * bits // 8, np.uint8)
    rc = lib().exl3c4_relayout(codes.ctypes.data, codes.shape[-1], rows, cols, bits, out.ctypes.data)
    if rc:
        raise ValueError(f"exl3c4_relayout: {STATUS.get(rc, rc)}")
    return out


def unrelayout(record: np.ndarray, rows: int, cols: int, bits: int) -> np.ndarray:
    record = np.ascontiguousarray(record, dtype=np.uint8)
    rb = (cols * bits + 7) // 8
    out = np.zeros((rows, rb), np.uint8)
    rc = lib().exl3c4_unrelayout(record.ctypes.data, rows, cols, bits, out.ctypes.data, rb)
    if rc:
        raise ValueError(f"exl3c4_unrelayout: {STATUS.get(rc, rc)}")
    return out


def record_to_codes(record: np.ndarray, rows: int, cols: int, bits: int) -> np.ndarray:
    """exllamav3's tile record (int16 [cols/16][rows/16][16 K]) -> canonical plane [rows][row_bytes]."""
    record = np.ascontiguousarray(record).view(np.uint16)
    rb = (cols * bits + 7) // 8
    out = np.zeros((rows, rb), np.uint8)
    rc = lib().exl3c4_record_to_codes(record.ctypes.data, rows, cols, bits, out.ctypes.data, rb)
    if rc:
        raise ValueError(f"exl3c4_record_to_codes: {STATUS.get(rc, rc)}")
    return out


# ------------------------------------------------------------------------------------------ the import (host)
class Checkpoint:
    """An EXL3 checkpoint directory opened for import (exl3c4_ckpt_open)."""

    def __init__(self, directory: str):
        self._h = None
        h = _p()
        rc = lib().exl3c4_ckpt_open(os.fsencode(directory), C.byref(h))
        if rc:
            raise OSError(rc, f"exl3c4_ckpt_open: {STATUS.get(rc, rc)}", directory)
        self._h = h

    @property
    def layers(self) -> int:
        return int(lib().exl3c4_ckpt_layers(self._h))

    def close(self):
        if self._h:
            lib().exl3c4_ckpt_close(self._h)
            self._h = None

    def __del__(self):
        self.close()

    def import_weight_rc(self, name: str, bits: int, cb, rows: int, cols: int, planes: dict) -> int:
        """exl3c4_import_weight into the caller's planes (numpy: codes uint8 [rows][row_bytes], suh / suh1 uint16 [cols],
        svh uint16 [rows]; suh1 None for a down weight): the status."""
        cb = CB[cb] if isinstance(cb, str) else cb
        codes = planes["codes"]
        s1 = planes.get("suh1")
        return lib().exl3c4_import_weight(self._h, name.encode(), bits, cb, rows, cols, codes.ctypes.data,
                                         codes.shape[1], planes["suh"].ctypes.data,
                                         None if s1 is None else s1.ctypes.data, planes["svh"].ctypes.data)

    def import_weight(self, name: str, bits: int, cb, rows: int, cols: int) -> dict:
        """The named routed-expert weight as canonical planes (a status other than OK raises)."""
        stacked = ".ffn_gate_up_exps." in name
        planes = {"codes": np.zeros((rows, (cols * bits + 7) // 8), np.uint8), "suh": np.zeros(cols, np.uint16),
                  "suh1": np.zeros(cols, np.uint16) if stacked else None, "svh": np.zeros(rows, np.uint16)}
        rc = self.import_weight_rc(name, bits, cb, rows, cols, planes)
        if rc:
            raise ValueError(f"exl3c4_import_weight({name}): {STATUS.get(rc, rc)}")
        return planes


def parse_weight_name(name: str):
    """(layer, expert, stacked) of a routed-expert weight name, or None (exl3c4_import_parse_name)."""
    layer, expert, stacked = _i32(), _i64(), _i32()
    rc = lib().exl3c4_import_parse_name(name.encode(), C.byref(layer), C.byref(expert), C.byref(stacked))
    return None if rc else (layer.value, expert.value, bool(stacked.value))


# ------------------------------------------------------------------------------------------ device calls
def _stream(stream):
    import torch
    s = torch.cuda.current_stream() if stream is None else stream
    return C.c_void_p(s.cuda_stream)


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def ptr(t):
    return _ptr(t)


def ctypes_ref(o: Op):
    return C.byref(o)


def stream_handle(stream=None):
    return _stream(stream)


# ------------------------------------------------------------------------------------------ HIP events (timing)
_hip = None


def hip():
    """The HIP runtime libexl3c4.so links, for events the caller owns (hipEventCreate / ElapsedTime)."""
    global _hip
    if _hip is None:
        lib()
        _hip = C.CDLL("libamdhip64.so")
        _hip.hipEventCreate.argtypes = [C.POINTER(_p)]
        _hip.hipEventElapsedTime.argtypes = [C.POINTER(C.c_float), _p, _p]
        _hip.hipEventDestroy.argtypes = [_p]
    return _hip


class Event:
    """A raw hipEvent_t (created at once, so a dispatch can stamp it)."""

    def __init__(self):
        self.h = _p()
        if hip().hipEventCreate(C.byref(self.h)):
            raise RuntimeError("hipEventCreate failed")

    def __del__(self):
        if _hip is not None and self.h:
            _hip.hipEventDestroy(self.h)


def elapsed_ms(a: Event, b: Event) -> float:
    ms = C.c_float()
    if hip().hipEventElapsedTime(C.byref(ms), a.h, b.h):
        raise RuntimeError("hipEventElapsedTime failed")
    return float(ms.value)


def launch_timed(o: Op, scratch, kernel: int, ev_start: Event, ev_stop: Event, stream=None) -> int:
    """exl3c4_launch with kernel `kernel` stamping ev_start / ev_stop at its own start and end."""
    n = 0 if scratch is None else scratch.numel()
    return int(lib().exl3c4_launch_timed(C.byref(o), _ptr(scratch), n, _stream(stream), kernel, ev_start.h,
                                         ev_stop.h))


def dequant(record, rows: int, cols: int, bits: int, cb, stream=None):
    """W_hat fp16 bits (torch.int16 [rows, cols]) of a stored record on the device."""
    import torch
    out = torch.empty((rows, cols), dtype=torch.int16, device=record.device)
    rc = lib().exl3c4_dequant(_ptr(record), rows, cols, bits, CB.get(cb, cb), _ptr(out), cols, _stream(stream))
    if rc:
        raise RuntimeError(f"exl3c4_dequant: {STATUS.get(rc, rc)}")
    return out


def prefill_min_rows(n_expert: int) -> int:
    """The least sorted-row count at which an op over n_expert experts takes the prefill path (exl3c4_prefill_min_rows)."""
    return int(lib().exl3c4_prefill_min_rows(n_expert))


def is_prefill(T: int, n_expert: int) -> bool:
    return T >= prefill_min_rows(n_expert)


def check_narrow(values, stream=None):
    """The device's own f32 -> bf16 and f32 -> f16 narrowing (the kernels' outputs' conversions) of a float32 device
    tensor: two uint16 numpy arrays (bf16 bits, f16 bits). A checker's entry (exl3c4_check_narrow)."""
    import torch
    n = values.numel()
    ob = torch.empty(n, dtype=torch.int16, device=values.device)
    oh = torch.empty(n, dtype=torch.int16, device=values.device)
    rc = lib().exl3c4_check_narrow(_ptr(values), _ptr(ob), _ptr(oh), n, _stream(stream))
    if rc:
        raise RuntimeError(f"exl3c4_check_narrow: {STATUS.get(rc, rc)}")
    torch.cuda.synchronize()
    return ob.cpu().numpy().view(np.uint16), oh.cpu().numpy().view(np.uint16)


def make_class(rows, cols, codes=None, suh=None, suh1=None, svh=None, dn_suh=None) -> Class:
    """One class's tables from STACKED device tensors ([entries, ...], contiguous entries)."""
    c = Class()
    c.rows, c.cols = rows, cols
    for name, t in (("codes", codes), ("suh", suh), ("suh1", suh1), ("svh", svh), ("dn_suh", dn_suh)):
        if t is None:
            setattr(c, name, None)
            setattr(c, name + "_stride", 0)
        else:
            setattr(c, name, t.data_ptr())
            setattr(c, name + "_stride", t.stride(0) * t.element_size())
    return c


def make_op(op, bits, cb, classes, x, sorted_tok, expert_offset, y, M, top_k, h_rot=0, a_rot=0, dn=None,
            x_bf16=False, n_expert=None, dn_bits=0) -> Op:
    o = Op()
    o.op, o.bits, o.codebook, o.dn_bits = op, bits, CB.get(cb, cb), dn_bits
    o.n_class, o.h_rot, o.a_rot = len(classes), h_rot, a_rot
    o.M, o.top_k = M, top_k
    o.n_expert = expert_offset.numel() - 1 if n_expert is None else n_expert
    for i, c in enumerate(classes):
        o.cls[i] = c
    for i, c in enumerate(dn or []):
        o.dn[i] = c
    o.x = x.data_ptr()
    o.x_dtype = BF16 if x_bf16 else F16
    o.x_rows, o.x_cols, o.x_pitch = x.shape[0], x.shape[1], x.stride(0)
    o.sorted_tok, o.expert_offset = sorted_tok.data_ptr(), expert_offset.data_ptr()
    o.y = y.data_ptr()
    o.T, o.y_cols, o.y_pitch = y.shape[0], y.shape[1], y.stride(0)
    return o


def scratch_bytes(o: Op) -> int:
    return int(lib().exl3c4_scratch_bytes(C.byref(o)))


def launch_scratch_bytes(o: Op) -> int:
    """The scratch this launch (its T rows) needs; exl3c4_launch refuses below it."""
    return int(lib().exl3c4_launch_scratch_bytes(C.byref(o)))


def launch(o: Op, scratch=None, stream=None) -> int:
    """Runs one op; returns the status (0 OK). `scratch`: a uint8 device tensor of >= scratch_bytes(o)."""
    n = 0 if scratch is None else scratch.numel()
    return int(lib().exl3c4_launch(C.byref(o), _ptr(scratch), n, _stream(stream)))


def launch_noalloc(o: Op, stream=None) -> int:
    """exl3c4_launch_noalloc: the launch in the library's own device scratch (no scratch argument, no allocation)."""
    return int(lib().exl3c4_launch_noalloc(C.byref(o), _stream(stream)))


def launch_checked(o: Op, scratch=None, stream=None) -> int:
    """launch, and a prefill-path launch also leaves its GEMMs' f32 sums in `scratch` for partial_sums."""
    n = 0 if scratch is None else scratch.numel()
    return int(lib().exl3c4_launch_checked(C.byref(o), _ptr(scratch), n, _stream(stream)))


def ctr_bytes(o: Op) -> int:
    """Bytes of the counter block exl3c4_launch_ctr takes for `o` (0: the op keeps no counters)."""
    return int(lib().exl3c4_ctr_bytes(C.byref(o)))


def launch_ctr(o: Op, scratch, ctr, stream=None) -> int:
    """exl3c4_launch_ctr: `ctr` a zeroed uint8 device tensor of >= ctr_bytes(o) bytes, 256-B aligned; left zeroed."""
    n = 0 if scratch is None else scratch.numel()
    m = 0 if ctr is None else ctr.numel()
    return int(lib().exl3c4_launch_ctr(C.byref(o), _ptr(scratch), n, _stream(stream), _ptr(ctr), m))


def launch_gather(o: Op, scratch, ctr, w, row_of, out, stream=None) -> int:
    """exl3c4_launch_gather: launch_ctr, then moe_gather of the op's y (bf16) into out (int16 bits [n_tok, cols], f16)
    with w f32 [n_tok, top_k] and row_of i32; the gather rides in gate_up_down's single kernel when it runs one."""
    n = 0 if scratch is None else scratch.numel()
    m = 0 if ctr is None else ctr.numel()
    return int(lib().exl3c4_launch_gather(C.byref(o), _ptr(scratch), n, _stream(stream), _ptr(ctr), m, _ptr(w),
                                          _ptr(row_of), _ptr(out), out.stride(0)))


def launch_leaving(o: Op, scratch, ctr, w, row_of, out, polls: int, stream=None) -> int:
    """exl3c4_launch_leaving: launch_gather, the single kernel's waiting down units leaving after `polls` polls."""
    n = 0 if scratch is None else scratch.numel()
    m = 0 if ctr is None else ctr.numel()
    return int(lib().exl3c4_launch_leaving(C.byref(o), _ptr(scratch), n, _stream(stream), _ptr(ctr), m, _ptr(w),
                                           _ptr(row_of), _ptr(out), out.stride(0), polls))


def partial_sums(o: Op, scratch, gemm: int = 0):
    """The f32 accumulations a launch left in `scratch` (torch tensor), splits added in the epilogue's order:
    float32 numpy [T, pitch]."""
    off, pitch, ss, n = _i64(), _i64(), _i64(), _i32()
    rc = lib().exl3c4_scratch_partials(C.byref(o), gemm, C.byref(off), C.byref(pitch), C.byref(ss), C.byref(n))
    if rc:
        raise RuntimeError(f"exl3c4_scratch_partials: {STATUS.get(rc, rc)}")
    raw = scratch.cpu().numpy()[off.value:].view(np.float32)
    T = o.T
    acc = raw[: T * pitch.value].reshape(T, pitch.value).copy()
    for s in range(1, n.value):      # columns no launch wrote hold whatever scratch held: no float warnings for them
        with np.errstate(over="ignore", invalid="ignore"):
            acc = (acc + raw[s * ss.value: s * ss.value + T * pitch.value].reshape(T, pitch.value)).astype(np.float32)
    return acc


def launch_status(o: Op, scratch) -> int:
    """The status word gate_up_down's single kernel left in `scratch` (0: good; 1: a wait gave up, the output is
    void), or None when the launch of `o` does not run that kernel."""
    off = _i64()
    if lib().exl3c4_scratch_status(C.byref(o), C.byref(off)):
        return None
    return int(scratch[off.value: off.value + 4].cpu().numpy().view(np.int32)[0])


# ------------------------------------------------------------------------------------------ the routing (device)
F32 = 2


_dtypes = {}


def _dt(t):
    if not _dtypes:
        import torch
        _dtypes.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    return _dtypes[t.dtype]


def router_topk(logits, top_k: int, renorm: bool = True, ids=None, w=None, stream=None) -> int:
    """exl3c4_router_topk on a device tensor [n_tok, n_expert] (f32 / f16 / bf16): fills ids (i32) and w (f32)
    [n_tok, top_k]; returns the status."""
    n_tok, n_expert = logits.shape
    return int(lib().exl3c4_router_topk(_ptr(logits), _dt(logits), n_tok, n_expert, logits.stride(0), top_k,
                                        int(renorm), _ptr(ids), _ptr(w), _stream(stream)))


def moe_scatter(ids, n_expert: int, sorted_tok, expert_offset, expert_count=None, row_of=None, expert_base: int = 0,
                stream=None) -> int:
    """exl3c4_moe_scatter on device i32 tensors: ids [n_tok, top_k] in; the rest out."""
    n_tok, top_k = ids.shape
    return int(lib().exl3c4_moe_scatter(_ptr(ids), n_tok, top_k, expert_base, n_expert, _ptr(sorted_tok),
                                        _ptr(expert_offset), _ptr(expert_count), _ptr(row_of), _stream(stream)))


def router_topk_scatter(logits, top_k: int, renorm: bool, ids, w, sorted_tok, expert_offset, expert_count=None,
                        row_of=None, stream=None) -> int:
    """exl3c4_router_topk_scatter: the router and the scatter in one call (one launch up to 16 tokens)."""
    n_tok, n_expert = logits.shape
    return int(lib().exl3c4_router_topk_scatter(_ptr(logits), _dt(logits), n_tok, n_expert, logits.stride(0), top_k,
                                                int(renorm), _ptr(ids), _ptr(w), _ptr(sorted_tok),
                                                _ptr(expert_offset), _ptr(expert_count), _ptr(row_of),
                                                _stream(stream)))


def moe_gather(y, y_bf16: bool, w, row_of, out, stream=None) -> int:
    """exl3c4_moe_gather: y int16 bits [T, cols] (bf16 or f16), w f32 [n_tok, top_k], row_of i32, out int16 bits
    [n_tok, cols] (f16)."""
    n_tok, top_k = w.shape
    return int(lib().exl3c4_moe_gather(_ptr(y), 1 if y_bf16 else 0, y.stride(0), _ptr(w), _ptr(row_of), n_tok, top_k,
                                       y.shape[1], _ptr(out), out.stride(0), _stream(stream)))


# ------------------------------------------------------------------------------------------ 16-bit and MX4 experts
def _launch_on(device, stream, fn, *args) -> int:
    """fn(*args, stream) with `device` current and, by default, on that device's current stream."""
    import torch
    if device.index == torch.cuda.current_device():
        return fn(*args, (torch.cuda.current_stream() if stream is None else stream).cuda_stream)
    with torch.cuda.device(device):
        return fn(*args, (torch.cuda.current_stream() if stream is None else stream).cuda_stream)


def _rows(t):
    """(rows, pitch in elements) of a tensor whose leading dimensions step evenly as one."""
    cols = t.shape[-1]
    if t.is_contiguous():
        return (t.numel() // cols if cols else 0), cols
    if cols > 1 and t.stride(-1) != 1:
        raise ValueError("rows have to be contiguous")
    rows, pitch = 1, None
    for d in range(t.dim() - 2, -1, -1):
        if t.shape[d] == 1:
            continue
        if pitch is None:
            pitch = t.stride(d)
        elif t.stride(d) != rows * pitch:
            raise ValueError("the leading dimensions do not step evenly: flatten them or call once for each")
        rows *= t.shape[d]
    return rows, cols if pitch is None else pitch


def mx4_empty(shape, device="cuda") -> Mx4:
    """Uninitialised MX4 rows for values of `shape` ([..., rows, cols])."""
    import torch
    *lead, cols = shape
    nb = (cols + 31) // 32
    return Mx4(torch.empty((*lead, 16 * nb), dtype=torch.uint8, device=device),
               torch.empty((*lead, (nb + 3) // 4 * 4), dtype=torch.uint8, device=device), cols)


_cuda = None                       # torch.cuda, from the first conversion on (an import statement a call is 0.1 us of 5)


def _convert(fn, v, q: Mx4, stream, quant: bool) -> int:
    """One of the conversions between the rows of v and q (a small one is bound by what happens here: rows that follow each
    other need no look at the strides)."""
    global _cuda
    if _cuda is None:
        import torch
        _cuda = torch.cuda
    dev = v.get_device()
    if v.shape != q.shape or dev != q.device:
        raise ValueError("the values and q have other shapes or devices")
    n, pitch = (q.rows, q.cols) if v.is_contiguous() else _rows(v)
    cp, sp = q._pitches or q.pitches()
    c, s, dt = q.codes.data_ptr(), q.scales.data_ptr(), _dtypes.get(v.dtype)
    if dt is None:
        dt = _dt(v)
    args = (v.data_ptr(), dt, n, q.cols, pitch, c, cp, s, sp) if quant else (c, cp, s, sp, n, q.cols, v.data_ptr(), dt, pitch)
    if stream is not None and dev == _cuda.current_device():
        return fn(*args, stream.cuda_stream)
    return _launch_on(v.device, stream, fn, *args)


def mx4_quant(x, q: Mx4, stream=None) -> int:
    """exl3c4_mx4_quant of x [..., cols] (f32 / f16 / bf16) into q; returns the status."""
    return _convert(lib().exl3c4_mx4_quant, x, q, stream, True)


def mx4_dequant(q: Mx4, out, stream=None) -> int:
    """exl3c4_mx4_dequant of q into out [..., cols] (f32 / f16 / bf16); returns the status."""
    return _convert(lib().exl3c4_mx4_dequant, out, q, stream, False)


def _planes(t):
    """(values or codes, scales or None, columns, type) of an operand of moe_gemm."""
    if isinstance(t, Mx4):
        return t.codes, t.scales, t.cols, MX4
    return t, None, t.shape[-1], _dt(t)


def make_gemm(x, w, sorted_tok, expert_offset, y, top_k: int = 1, act: int = ACT_NONE) -> Gemm:
    """One moe_gemm: x [x_rows, K] and w [n_expert, N, K], each a 16-bit tensor or Mx4, sorted_tok i32 [T] (None: x holds
    sorted rows), expert_offset i32 [n_expert + 1], y [T, N] ([T, N / 2] with ACT_SWIGLU) f16, bf16 or f32."""
    xv, xs, K, xt = _planes(x)
    wv, ws, Kw, wt = _planes(w)
    if xv.dim() != 2 or wv.dim() != 3 or y.dim() != 2:
        raise ValueError("x and y are rows, w one [N, K] an expert")
    g = Gemm()
    g.x_type, g.w_type, g.y_type, g.act = xt, wt, _dt(y), act
    E, N = wv.shape[0], wv.shape[1]
    g.N, g.K, g.n_expert, g.top_k, g.T = N, K, E, top_k, y.shape[0]
    if Kw != K or y.shape[1] != (N // 2 if act == ACT_SWIGLU else N) or \
            expert_offset.numel() < E + 1:
        raise ValueError("x, w, expert_offset and y do not fit together")
    for t, n in ((sorted_tok, g.T), (expert_offset, E + 1)):
        if t is not None and (t.element_size() != 4 or t.is_floating_point() or not t.is_contiguous() or t.numel() < n):
            raise ValueError("sorted_tok and expert_offset are contiguous int32, of T and n_expert + 1 values at least")
    for t in (xv, xs, wv, ws, y):
        if t is not None and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError("rows have to be contiguous")
    for t in (xv, xs, wv, ws, sorted_tok, expert_offset):
        if t is not None and t.device != y.device:
            raise ValueError("the operands are on other devices")
    for t in (wv, ws):                                         # a stride of 0 would name a pointer array
        if t is not None and E > 1 and t.stride(0) == 0:
            raise ValueError("the experts' weights are one: pass n_expert 1")

    def pitch(t, d):                                           # of one row alone: any that is large enough
        return t.stride(d) if t.shape[d] > 1 else max(t.stride(d), t.shape[-1])

    def stride(t):
        return (t.stride(0) if E > 1 else N * pitch(t, 1)) * t.element_size()
    g.x, g.x_rows, g.x_pitch = xv.data_ptr(), xv.shape[0], pitch(xv, 0)
    g.w, g.w_pitch, g.w_stride = wv.data_ptr(), pitch(wv, 1), stride(wv)
    if xs is not None:
        g.x_scales, g.xs_pitch = xs.data_ptr(), pitch(xs, 0)
    if ws is not None:
        g.w_scales, g.ws_pitch, g.ws_stride = ws.data_ptr(), pitch(ws, 1), stride(ws)
    g.sorted_tok = None if sorted_tok is None else sorted_tok.data_ptr()
    g.expert_offset, g.y, g.y_pitch = expert_offset.data_ptr(), y.data_ptr(), pitch(y, 0)
    g.device, g.tensors = y.device, (xv, xs, wv, ws, sorted_tok, expert_offset, y)     # alive as long as g
    return g


def moe_gemm(g: Gemm, stream=None) -> int:
    """exl3c4_moe_gemm on the device of g's tensors; returns the status."""
    return _launch_on(g.device, stream, lib().exl3c4_moe_gemm, C.byref(g))


def alloc_scratch(o: Op, device="cuda"):
    import torch
    n = scratch_bytes(o)
    if n < 0:
        raise RuntimeError(f"exl3c4_scratch_bytes: {STATUS.get(n, n)}")
    return torch.empty(max(n, 256), dtype=torch.uint8, device=device)
