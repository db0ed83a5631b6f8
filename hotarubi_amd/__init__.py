"""hotarubi_amd -- MI355X (gfx950) backend for hotarubi's GEMM instruction.

Python host mirror of the reference interface, over the C ABI in
include/hotarubi_gpu.h (libhotarubi_gpu.so, built by hotarubi_amd.build):

  GemmCommand / VecCommand   field for field iss::GemmCommand, iss::VecCommand
                             (tools/iss/gemm_array.hpp:16-27,
                              tools/iss/vec_engine.hpp:70-81)
  DeviceMemories             device copies of iss::Memories
                             (tools/iss/memories.hpp:86-96), ISS word layout
  execute_gemm(cmd, mem)     iss::ExecuteGemm (tools/iss/gemm_array.cpp:112)
  vec_execute(cmd, mem)      VecEngine::Execute for library entries 0-9
  linear(...)                a linear layer as LinearEmitter::Emit emits it
                             (tools/compiler/kernels.cpp:343-395) + epilogue
  encode_mxint8(x)           EncodeMxint8 + PackAbuf (formats.cpp:114-162)
  kv_plan, norm_rope, kv_append, kv_read, kv_attention
                             a serving step's attention over a paged MXFP4
                             cache (torch tensors; no counterpart)
  kv_attention_way           how kv_attention would divide a call's work
  kv8_append, kv8_read, kv8_attention, kv8_attention_way
                             the same over a paged cache of 8 bits
  kv_fork, kv_copy, kv_free, kv_compact
                             pages that requests share, give back and move
  token_logprobs             log probabilities, entropy and the most likely
                             tokens of a step's logits

Errors raise HbError; a command the reference rejects with Fail raises
HbBadCommand carrying the reference's message.  The library is loaded from
this directory and the package fails loudly when it is missing: there is no
CPU fallback.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
import threading
from dataclasses import dataclass, fields

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libhotarubi_gpu.so")

HB_OK, HB_EBADCMD, HB_EINVAL, HB_EUNSUPPORTED, HB_EDEVICE, HB_ENOMEM = range(6)
ABUF, WBUF, FBUF, PBUF, TBUF = range(5)
DEPTH = {ABUF: 8192, WBUF: 2048, FBUF: 4096, PBUF: 512, TBUF: 1024}
WORD_BYTES = {ABUF: 132, WBUF: 144, FBUF: 128, PBUF: 128, TBUF: 8}
EXACT, FAST = 0, 1
PANELS = 2  # hb_linear_desc.flags bit: the W planes are weight panels
W8_PANELS = 4  # flags bit: a W8 layer's planes are W8 panels (w[0] = w[1])
A_FP8 = 8  # flags bit: A holds MXFP8 E4M3 codes (hb_encode_mxfp8), one MXFP4 plane
EP_ADDP, EP_MULP, EP_SCALE, EP_COPY, EP_RELU, EP_ACT, EP_ACT_MUL = 3, 4, 5, 6, 7, 8, 9
EP_ADD = 0x100
MAX_PIECES, MAX_OPS = 16, 8
ABI_VERSION = 3  # HB_ABI_VERSION of the structs mirrored below

#: every symbol include/hotarubi_gpu.h declares
EXPORTS = (
    "hb_abi_version", "hb_last_error", "hb_ctx_create", "hb_ctx_destroy",
    "hb_ctx_set_stream", "hb_ctx_synchronize", "hb_onchip_create", "hb_onchip_destroy",
    "hb_onchip_upload", "hb_onchip_download", "hb_onchip_device_ptr", "hb_gemm_decode",
    "hb_gemm_encode", "hb_gemm_check", "hb_gemm_access", "hb_gemm_exec", "hb_gemm_exec_async",
    "hb_gemm_cycles", "hb_vec_exec", "hb_linear", "hb_linear_async",
    "hb_linear_batched_async", "hb_encode_mxint8", "hb_encode_mxfp8", "hb_split8",
    "hb_split8_async",
    "hb_t32_split8", "hb_t32_split8_async", "hb_rows", "hb_rows_async",
    "hb_row_load", "hb_row_load_async", "hb_row_store", "hb_row_store_async",
    "hb_gacc", "hb_gacc_async", "hb_panel_bytes", "hb_pack_weights", "hb_unpack_weights",
    "hb_linear_noalloc_async", "hb_w8_panel_bytes", "hb_pack_w8", "hb_unpack_w8",
    "hb_w8_from_fp32", "hb_mxfp4_canonical", "hb_image_create", "hb_image_destroy",
    "hb_image_alloc", "hb_image_set_reuse", "hb_image_define", "hb_image_put", "hb_image_get",
    "hb_image_region", "hb_image_region_count", "hb_image_region_at", "hb_image_end",
    "hb_image_base", "hb_linear_group_async",
    "hb_kv_plan", "hb_kv_plan_async", "hb_norm_rope", "hb_norm_rope_async", "hb_kv_append",
    "hb_kv_append_async", "hb_kv_read", "hb_kv_read_async", "hb_kv_attention",
    "hb_kv_attention_async", "hb_kv_attention_way",
    "hb_kv8_append", "hb_kv8_append_async", "hb_kv8_read", "hb_kv8_read_async",
    "hb_kv8_attention", "hb_kv8_attention_async", "hb_kv8_attention_way",
    "hb_kv_fork", "hb_kv_fork_async", "hb_kv_copy", "hb_kv_copy_async", "hb_kv_free",
    "hb_kv_free_async", "hb_kv_compact", "hb_kv_compact_async", "hb_token_logprobs",
    "hb_token_logprobs_async",
)


class HbError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"[{code}] {message}")
        self.code = code
        self.message = message


class HbBadCommand(HbError):
    """A command the reference rejects (Require -> Fail)."""


class _GemmCmd(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in
                ("a_base", "a_stride", "kb", "m", "w_base", "w_stride", "n8", "c_base",
                 "wmode", "acc")]


class _VecCmd(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in
                ("entry", "quantize", "src", "src2", "dst", "rows_q", "n8", "p_base", "aux",
                 "imm")]


class _Piece(C.Structure):
    _fields_ = [("kb_offset", C.c_uint32), ("kb", C.c_uint32), ("a_word", C.c_uint32)]


class _EpOp(C.Structure):
    _fields_ = [("op", C.c_uint32), ("imm", C.c_uint32), ("vec", C.c_void_p),
                ("x2", C.c_void_p)]


class _RowsDesc(C.Structure):
    _fields_ = [("entry", C.c_uint32), ("rows", C.c_uint32), ("cols", C.c_uint32),
                ("aux", C.c_uint32), ("imm", C.c_uint32), ("x", C.c_void_p),
                ("gamma", C.c_void_p), ("beta", C.c_void_p), ("tbuf", C.c_void_p),
                ("y", C.c_void_p), ("q_out", C.c_void_p)]


class _GaccDesc(C.Structure):
    _fields_ = [("base", C.c_void_p), ("list", C.c_void_p), ("list_stride", C.c_uint64),
                ("quads", C.c_uint32), ("slots", C.c_uint32), ("blocks", C.c_uint32),
                ("w_stride", C.c_uint32), ("accumulate", C.c_uint32), ("out", C.c_void_p)]


class _LinearDesc(C.Structure):
    _fields_ = [("m", C.c_uint32), ("n", C.c_uint32), ("kb_total", C.c_uint32),
                ("n_planes", C.c_uint32), ("modes", C.c_uint32 * 2), ("a", C.c_void_p),
                ("w", C.c_void_p * 2), ("n_pieces", C.c_uint32),
                ("pieces", _Piece * MAX_PIECES), ("onto", C.c_uint32), ("c", C.c_void_p),
                ("n_ops", C.c_uint32), ("ops", _EpOp * MAX_OPS), ("tbuf", C.c_void_p),
                ("q_out", C.c_void_p), ("flags", C.c_uint32), ("a_stride", C.c_uint32)]


@dataclass
class GemmCommand:
    """iss::GemmCommand (tools/iss/gemm_array.hpp:16-27)."""

    a_base: int = 0
    a_stride: int = 0
    kb: int = 0
    m: int = 0
    w_base: int = 0
    w_stride: int = 0
    n8: int = 0
    c_base: int = 0
    wmode: int = 0
    acc: bool = False

    def _c(self) -> _GemmCmd:
        return _GemmCmd(*[int(getattr(self, f.name)) for f in fields(self)])


@dataclass
class VecCommand:
    """iss::VecCommand (tools/iss/vec_engine.hpp:70-81)."""

    entry: int = 0
    quantize: bool = False
    src: int = 0
    src2: int = 0
    dst: int = 0
    rows_q: int = 0
    n8: int = 0
    p_base: int = 0
    aux: int = 0
    imm: int = 0

    def _c(self) -> _VecCmd:
        return _VecCmd(*[int(getattr(self, f.name)) for f in fields(self)])


_lib = None


def lib():
    """Load libhotarubi_gpu.so; raises if it was not built (no fallback)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: run `python -m hotarubi_amd.build`")
        L = C.CDLL(LIB_PATH)
        vp, u32, i = C.c_void_p, C.c_uint32, C.c_int
        sig = {
            "hb_abi_version": (i, []),
            "hb_last_error": (C.c_char_p, []),
            "hb_ctx_create": (i, [i, C.POINTER(vp)]),
            "hb_ctx_destroy": (i, [vp]),
            "hb_ctx_set_stream": (i, [vp, vp]),
            "hb_ctx_synchronize": (i, [vp]),
            "hb_onchip_create": (i, [vp, C.POINTER(vp)]),
            "hb_onchip_destroy": (i, [vp]),
            "hb_onchip_upload": (i, [vp, i, u32, u32, vp]),
            "hb_onchip_download": (i, [vp, i, u32, u32, vp]),
            "hb_onchip_device_ptr": (i, [vp, i, C.POINTER(vp)]),
            "hb_gemm_decode": (i, [vp, C.POINTER(_GemmCmd)]),
            "hb_gemm_encode": (i, [C.POINTER(_GemmCmd), vp]),
            "hb_gemm_check": (i, [C.POINTER(_GemmCmd)]),
            "hb_gemm_access": (i, [C.POINTER(_GemmCmd), vp, vp, vp, vp]),
            "hb_gemm_exec": (i, [vp, C.POINTER(_GemmCmd), vp]),
            "hb_gemm_exec_async": (i, [vp, C.POINTER(_GemmCmd), vp]),
            "hb_gemm_cycles": (C.c_uint64, [C.POINTER(_GemmCmd), u32]),
            "hb_vec_exec": (i, [vp, C.POINTER(_VecCmd), vp]),
            "hb_linear": (i, [vp, C.POINTER(_LinearDesc)]),
            "hb_linear_async": (i, [vp, C.POINTER(_LinearDesc)]),
            "hb_linear_batched_async": (i, [vp, C.POINTER(_LinearDesc), u32]),
            "hb_linear_group_async": (i, [vp, C.POINTER(_LinearDesc), u32]),
            "hb_linear_noalloc_async": (i, [vp, C.POINTER(_LinearDesc), u32]),
            "hb_encode_mxint8": (i, [vp, vp, u32, u32, vp]),
            "hb_encode_mxfp8": (i, [vp, vp, u32, u32, vp]),
            "hb_gacc": (i, [vp, C.POINTER(_GaccDesc)]),
            "hb_gacc_async": (i, [vp, C.POINTER(_GaccDesc)]),
            "hb_row_load": (i, [vp, vp, C.c_uint64, u32, u32, u32, vp, vp]),
            "hb_row_load_async": (i, [vp, vp, C.c_uint64, u32, u32, u32, vp, vp]),
            "hb_row_store": (i, [vp, vp, u32, u32, u32, vp, C.c_uint64]),
            "hb_row_store_async": (i, [vp, vp, u32, u32, u32, vp, C.c_uint64]),
            "hb_rows": (i, [vp, C.POINTER(_RowsDesc)]),
            "hb_rows_async": (i, [vp, C.POINTER(_RowsDesc)]),
            "hb_split8": (i, [vp, vp, C.c_uint64, u32, u32, vp, vp]),
            "hb_split8_async": (i, [vp, vp, C.c_uint64, u32, u32, vp, vp]),
            "hb_t32_split8": (i, [vp, vp, C.c_uint64, u32, u32, vp, vp]),
            "hb_t32_split8_async": (i, [vp, vp, C.c_uint64, u32, u32, vp, vp]),
            "hb_panel_bytes": (C.c_uint64, [u32, u32]),
            "hb_pack_weights": (i, [vp, vp, u32, u32, vp]),
            "hb_unpack_weights": (i, [vp, vp, u32, u32, vp]),
            "hb_w8_panel_bytes": (C.c_uint64, [u32, u32]),
            "hb_pack_w8": (i, [vp, vp, vp, u32, u32, vp]),
            "hb_unpack_w8": (i, [vp, vp, u32, u32, vp, vp]),
            "hb_w8_from_fp32": (i, [vp, vp, u32, u32, u32, vp, vp]),
            "hb_mxfp4_canonical": (i, [vp, vp, vp, u32, u32, C.c_int32, u32, vp]),
            "hb_image_create": (i, [vp, C.c_uint64, C.POINTER(vp)]),
            "hb_image_destroy": (None, [vp]),
            "hb_image_alloc": (i, [vp, C.c_char_p, C.c_uint64, C.c_uint64,
                                   C.POINTER(C.c_uint64)]),
            "hb_image_set_reuse": (None, [vp, i]),
            "hb_image_define": (i, [vp, C.c_char_p, C.c_uint64, C.c_uint64]),
            "hb_image_put": (i, [vp, C.c_uint64, vp, C.c_uint64]),
            "hb_image_get": (i, [vp, C.c_uint64, vp, C.c_uint64]),
            "hb_image_region": (i, [vp, C.c_char_p, C.POINTER(C.c_uint64),
                                    C.POINTER(C.c_uint64)]),
            "hb_image_region_count": (u32, [vp]),
            "hb_image_region_at": (i, [vp, u32, C.POINTER(C.c_char_p), C.POINTER(C.c_uint64),
                                       C.POINTER(C.c_uint64)]),
            "hb_image_end": (C.c_uint64, [vp]),
            "hb_image_base": (vp, [vp]),
            "hb_kv_plan": (i, [vp, vp]),
            "hb_kv_plan_async": (i, [vp, vp]),
            "hb_norm_rope": (i, [vp, vp]),
            "hb_norm_rope_async": (i, [vp, vp]),
            "hb_kv_append": (i, [vp, vp]),
            "hb_kv_append_async": (i, [vp, vp]),
            "hb_kv_read": (i, [vp, vp]),
            "hb_kv_read_async": (i, [vp, vp]),
            "hb_kv_attention": (i, [vp, vp]),
            "hb_kv_attention_async": (i, [vp, vp]),
            "hb_kv_attention_way": (i, [vp, vp]),
            "hb_kv8_attention_way": (i, [vp, vp]),
            "hb_kv8_append": (i, [vp, vp]),
            "hb_kv8_append_async": (i, [vp, vp]),
            "hb_kv8_read": (i, [vp, vp]),
            "hb_kv8_read_async": (i, [vp, vp]),
            "hb_kv8_attention": (i, [vp, vp]),
            "hb_kv8_attention_async": (i, [vp, vp]),
            "hb_kv_fork": (i, [vp, vp]),
            "hb_kv_fork_async": (i, [vp, vp]),
            "hb_kv_copy": (i, [vp, vp]),
            "hb_kv_copy_async": (i, [vp, vp]),
            "hb_kv_free": (i, [vp, vp]),
            "hb_kv_free_async": (i, [vp, vp]),
            "hb_kv_compact": (i, [vp, vp]),
            "hb_kv_compact_async": (i, [vp, vp]),
            "hb_token_logprobs": (i, [vp, vp]),
            "hb_token_logprobs_async": (i, [vp, vp]),
        }
        for name, (res, args) in sig.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        if L.hb_abi_version() != ABI_VERSION:
            raise ImportError(f"{LIB_PATH} has ABI {L.hb_abi_version()}, this module {ABI_VERSION}: "
                              "rebuild with `python -m hotarubi_amd.build`")
        _lib = L
    return _lib


def last_error() -> str:
    return lib().hb_last_error().decode()


def _check(rc: int) -> None:
    if rc != HB_OK:
        cls = HbBadCommand if rc == HB_EBADCMD else HbError
        raise cls(rc, last_error())


# ------------------------------------------------------------- context --

class Context:
    """hb_ctx: one per host thread, owns a HIP stream on `device`."""

    def __init__(self, device: int = 0):
        h = C.c_void_p()
        _check(lib().hb_ctx_create(device, C.byref(h)))
        self.handle = h
        self.device = device

    def close(self):
        if self.handle:
            lib().hb_ctx_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def synchronize(self):
        _check(lib().hb_ctx_synchronize(self.handle))

    def set_stream(self, stream_ptr: int | None):
        _check(lib().hb_ctx_set_stream(self.handle, stream_ptr))


_default_ctx = None


def default_context() -> Context:
    global _default_ctx
    if _default_ctx is None:
        _default_ctx = Context(0)
    return _default_ctx


class DeviceMemories:
    """Device copies of the on-chip memories in the ISS word layout."""

    def __init__(self, ctx: Context | None = None):
        self.ctx = ctx or default_context()
        h = C.c_void_p()
        _check(lib().hb_onchip_create(self.ctx.handle, C.byref(h)))
        self.handle = h

    def close(self):
        if self.handle:
            lib().hb_onchip_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def upload(self, mem: int, array: np.ndarray, first: int = 0) -> None:
        a = np.ascontiguousarray(array)
        count = a.nbytes // WORD_BYTES[mem]
        if count * WORD_BYTES[mem] != a.nbytes:
            raise ValueError("array is not a whole number of words")
        _check(lib().hb_onchip_upload(self.handle, mem, first, count, a.ctypes.data))

    def download(self, mem: int, first: int = 0, count: int | None = None) -> np.ndarray:
        count = DEPTH[mem] - first if count is None else count
        out = np.zeros(count * WORD_BYTES[mem], np.uint8)
        _check(lib().hb_onchip_download(self.handle, mem, first, count, out.ctypes.data))
        shape = {ABUF: (count, 132), WBUF: (count, 144)}.get(mem)
        if shape:
            return out.reshape(shape)
        if mem == TBUF:
            return out.view(np.uint64)
        return out.view(np.uint32).reshape(count, 32)

    def upload_all(self, abuf=None, wbuf=None, fbuf=None, pbuf=None, tbuf=None):
        for mem, arr in ((ABUF, abuf), (WBUF, wbuf), (FBUF, fbuf), (PBUF, pbuf), (TBUF, tbuf)):
            if arr is not None:
                self.upload(mem, arr)

    def device_ptr(self, mem: int) -> int:
        p = C.c_void_p()
        _check(lib().hb_onchip_device_ptr(self.handle, mem, C.byref(p)))
        return p.value


# ---------------------------------------------------- instruction level --

def decode_gemm(word: bytes) -> GemmCommand:
    """DecodeGemm (tools/iss/machine.cpp:93-104) of a 16-byte instruction."""
    buf = (C.c_uint8 * 16).from_buffer_copy(bytes(word))
    cmd = _GemmCmd()
    _check(lib().hb_gemm_decode(buf, C.byref(cmd)))
    return GemmCommand(*[getattr(cmd, f.name) for f in fields(GemmCommand)])


def encode_gemm(cmd: GemmCommand) -> bytes:
    buf = (C.c_uint8 * 16)()
    _check(lib().hb_gemm_encode(C.byref(cmd._c()), buf))
    return bytes(buf)


def check_gemm(cmd: GemmCommand) -> None:
    _check(lib().hb_gemm_check(C.byref(cmd._c())))


def gemm_access(cmd: GemmCommand):
    ra = np.zeros(8192, np.uint8)
    rw = np.zeros(2048, np.uint8)
    rf = np.zeros(4096, np.uint8)
    wf = np.zeros(4096, np.uint8)
    _check(lib().hb_gemm_access(C.byref(cmd._c()), ra.ctypes.data, rw.ctypes.data,
                                rf.ctypes.data, wf.ctypes.data))
    return ra, rw, rf, wf


def gemm_cycles(cmd: GemmCommand, fixed_cycles: int = 51) -> int:
    return int(lib().hb_gemm_cycles(C.byref(cmd._c()), fixed_cycles))


def execute_gemm(cmd: GemmCommand, mem: DeviceMemories, sync: bool = True) -> None:
    """iss::ExecuteGemm on the device images (bit-exact)."""
    f = lib().hb_gemm_exec if sync else lib().hb_gemm_exec_async
    _check(f(mem.ctx.handle, C.byref(cmd._c()), mem.handle))


def vec_execute(cmd: VecCommand, mem: DeviceMemories) -> None:
    """VecEngine::Execute for library entries 0-9 (bit-exact)."""
    _check(lib().hb_vec_exec(mem.ctx.handle, C.byref(cmd._c()), mem.handle))


# -------------------------------------------------------- linear level --

def _ptr(t) -> int | None:
    """Device address of a torch tensor (or an int address, or None)."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def linear_desc(m, n, kb_total, a, planes, modes, c, pieces=None, onto=False, ops=(),
                tbuf=None, q_out=None, mode=EXACT, a_stride=0, panels=False,
                w8_panels=False, a_fp8=False) -> _LinearDesc:
    """Build an hb_linear_desc from device buffers (torch tensors or addresses).

    planes/modes: [w] with [0] (FP4) or [w_hi, w_lo] with [1, 2] (W8);
    w8_panels: planes = [p, p] for the W8 panels p of hb_pack_w8.
    a_fp8: A holds MXFP8 E4M3 words (hb_encode_mxfp8); planes = [w], modes [0].
    pieces: (kb_offset, kb) or, with a_stride (A words per quad) nonzero,
    (kb_offset, kb, a_word): LinearPiece (kernels.hpp:69-74) with its A
    place as a word offset from `a`.
    ops: sequence of (kind, arg): ADDP/MULP take a device vector, SCALE an FP32
    bit pattern, ACT_MUL/ADD a device [m][n] tensor, COPY/RELU/ACT None.
    """
    d = _LinearDesc()
    d.m, d.n, d.kb_total = m, n, kb_total
    d.n_planes = len(planes)
    for i, (w, md) in enumerate(zip(planes, modes)):
        d.w[i] = _ptr(w)
        d.modes[i] = md
    d.a = _ptr(a)
    pieces = pieces or [(0, kb_total)]
    if len(pieces) > MAX_PIECES:
        raise ValueError("too many pieces")
    d.n_pieces = len(pieces)
    for i, pc in enumerate(pieces):
        off, kb = pc[0], pc[1]
        d.pieces[i] = _Piece(off, kb, pc[2] if len(pc) > 2 else 0)
    d.a_stride = a_stride
    d.onto = 1 if onto else 0
    d.c = _ptr(c)
    if len(ops) > MAX_OPS:
        raise ValueError("too many ops")
    d.n_ops = len(ops)
    for i, (kind, arg) in enumerate(ops):
        d.ops[i].op = kind
        if kind in (EP_ADDP, EP_MULP):
            d.ops[i].vec = _ptr(arg)
        elif kind == EP_SCALE:
            d.ops[i].imm = int(arg)
        elif kind in (EP_ACT_MUL, EP_ADD):
            d.ops[i].x2 = _ptr(arg)
    d.tbuf = _ptr(tbuf)
    d.q_out = _ptr(q_out)
    d.flags = mode | (PANELS if panels else 0) | (W8_PANELS if w8_panels else 0) | \
        (A_FP8 if a_fp8 else 0)
    return d


def linear(ctx: Context | None = None, sync: bool = True, **kw) -> None:
    ctx = ctx or default_context()
    d = linear_desc(**kw)
    f = lib().hb_linear if sync else lib().hb_linear_async
    _check(f(ctx.handle, C.byref(d)))


def launch(desc: _LinearDesc, ctx: Context | None = None) -> None:
    """hb_linear_async on a prebuilt descriptor (ordered on the context's stream)."""
    ctx = ctx or default_context()
    _check(lib().hb_linear_async(ctx.handle, C.byref(desc)))


def linear_group(descs, ctx: Context | None = None) -> None:
    """hb_linear_group_async: up to 4 independent small fast layers (and
    gated pairs) in one launch where possible; the result of launching them
    in order.  descs: a list of descriptors or a prebuilt ctypes array of
    them (reused across calls)."""
    ctx = ctx or default_context()
    arr = descs if isinstance(descs, C.Array) else (_LinearDesc * len(descs))(*descs)
    _check(lib().hb_linear_group_async(ctx.handle, arr, len(descs)))


def linear_batched(descs, ctx: Context | None = None) -> None:
    ctx = ctx or default_context()
    arr = (_LinearDesc * len(descs))(*descs)
    _check(lib().hb_linear_batched_async(ctx.handle, arr, len(descs)))


def linear_noalloc(descs, ctx: Context | None = None) -> None:
    """hb_linear_noalloc_async: hb_linear_batched_async without any device
    allocation (the K-split scratch is a fixed per-device array)."""
    ctx = ctx or default_context()
    arr = (_LinearDesc * len(descs))(*descs)
    _check(lib().hb_linear_noalloc_async(ctx.handle, arr, len(descs)))


NOALLOC_SCRATCH_BYTES = 8 << 20  # HB_NOALLOC_SCRATCH_BYTES


def gacc(base, lst, quads: int, slots: int, blocks: int, w_stride: int, out,
         list_stride: int = 0, accumulate: bool = False, ctx: Context | None = None,
         sync: bool = True) -> None:
    """hb_gacc: the DMA engine's gather-accumulate (dma_engine.cpp:596-656)
    over `quads` quads' lists, into out fp32 [quads * 4][32 * blocks]."""
    ctx = ctx or default_context()
    d = _GaccDesc(_ptr(base), _ptr(lst), list_stride, quads, slots, blocks, w_stride,
                  1 if accumulate else 0, _ptr(out))
    fn = lib().hb_gacc if sync else lib().hb_gacc_async
    _check(fn(ctx.handle, C.byref(d)))


def row_token_bytes(tok: int) -> int:
    """Bytes of one MXINT8 token in the DMA row format."""
    return (2 * tok + (2 if tok > 16 else 1)) * 16


def row_load(src, rows: int, row_words: int, tok: int, out, row_stride: int | None = None,
             index=None, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_row_load: DMA_LD ROW / ROW_INDEXED (dma_engine.cpp:218-244) of MXINT8
    tokens into DDR A words [rows * row_words / 4][tok] x 144 B."""
    ctx = ctx or default_context()
    stride = row_words * row_token_bytes(tok) if row_stride is None else row_stride
    fn = lib().hb_row_load if sync else lib().hb_row_load_async
    _check(fn(ctx.handle, _ptr(src), stride, rows, row_words, tok, _ptr(index), _ptr(out)))


def row_store(words, rows: int, row_words: int, tok: int, dst, row_stride: int | None = None,
              ctx: Context | None = None, sync: bool = True) -> None:
    """hb_row_store: DMA_ST ROW (dma_engine.cpp:262-279), A words -> tokens."""
    ctx = ctx or default_context()
    stride = row_words * row_token_bytes(tok) if row_stride is None else row_stride
    fn = lib().hb_row_store if sync else lib().hb_row_store_async
    _check(fn(ctx.handle, _ptr(words), rows, row_words, tok, _ptr(dst), stride))


ROWS_SOFTMAX, ROWS_LAYERNORM, ROWS_RMSNORM = 12, 22, 34


def rows(entry: int, x, rows: int, cols: int, aux: int, imm: int = 0, gamma=None, beta=None,
         tbuf=None, y=None, q_out=None, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_rows: a VEC row program (12 SOFTMAX, 22 LAYERNORM, 34 RMSNORM;
    vec_rom.cpp:133-212, 239-272) over fp32 [rows][cols] device rows, into y
    (fp32) or q_out (MXINT8 DDR words, the A of `linear`)."""
    ctx = ctx or default_context()
    d = _RowsDesc(entry, rows, cols, aux, imm, _ptr(x), _ptr(gamma), _ptr(beta), _ptr(tbuf),
                  _ptr(y), _ptr(q_out))
    fn = lib().hb_rows if sync else lib().hb_rows_async
    _check(fn(ctx.handle, C.byref(d)))


def panel_bytes(n: int, kb_total: int) -> int:
    """Bytes of one weight plane in the panel layout (hb_panel_bytes)."""
    return int(lib().hb_panel_bytes(n, kb_total))


def pack_weights(w, n: int, kb_total: int, panels, ctx: Context | None = None) -> None:
    """hb_pack_weights: DDR words [n/8][kb_total] x 144 B -> weight panels."""
    ctx = ctx or default_context()
    _check(lib().hb_pack_weights(ctx.handle, _ptr(w), n, kb_total, _ptr(panels)))


def unpack_weights(panels, n: int, kb_total: int, w, ctx: Context | None = None) -> None:
    """hb_unpack_weights: weight panels -> DDR words, bit for bit."""
    ctx = ctx or default_context()
    _check(lib().hb_unpack_weights(ctx.handle, _ptr(panels), n, kb_total, _ptr(w)))


def w8_panel_bytes(n: int, kb_total: int) -> int:
    """Bytes of a W8 layer's W8 panels (hb_w8_panel_bytes)."""
    return int(lib().hb_w8_panel_bytes(n, kb_total))


def pack_w8(w_hi, w_lo, n: int, kb_total: int, panels, ctx: Context | None = None) -> None:
    """hb_pack_w8: a W8 layer's hi and lo DDR word planes -> W8 panels."""
    ctx = ctx or default_context()
    _check(lib().hb_pack_w8(ctx.handle, _ptr(w_hi), _ptr(w_lo), n, kb_total, _ptr(panels)))


def unpack_w8(panels, n: int, kb_total: int, w_hi, w_lo, ctx: Context | None = None) -> None:
    """hb_unpack_w8: W8 panels -> the hi and lo DDR word planes, bit for bit."""
    ctx = ctx or default_context()
    _check(lib().hb_unpack_w8(ctx.handle, _ptr(panels), n, kb_total, _ptr(w_hi), _ptr(w_lo)))


def w8_from_fp32(w, rows: int, cols: int, out_rows: int, w_hi, w_lo,
                 ctx: Context | None = None) -> None:
    """hb_w8_from_fp32: fp32 weights [rows][cols] -> the W8 hi and lo WBUF word
    planes [out_rows/8][ceil(cols/32)] x 144 B (PadRows, EncodeMxint8, SplitW8,
    PackWbuf)."""
    ctx = ctx or default_context()
    _check(lib().hb_w8_from_fp32(ctx.handle, _ptr(w), rows, cols, out_rows, _ptr(w_hi),
                                 _ptr(w_lo)))


def mxfp4_canonical(codes, scales, rows: int, cols: int, out_rows: int, w,
                    exponent_shift: int = 0, ctx: Context | None = None) -> None:
    """hb_mxfp4_canonical: MXFP4 codes [rows][cols] and E8M0 scale bytes
    [rows][cols/32] -> canonical WBUF words [out_rows/8][cols/32] x 144 B
    (CanonicalMxfp4, PackWbuf)."""
    ctx = ctx or default_context()
    _check(lib().hb_mxfp4_canonical(ctx.handle, _ptr(codes), _ptr(scales), rows, cols,
                                    exponent_shift, out_rows, _ptr(w)))


class Image:
    """hb_image: the compiler's DDR image container (DdrImage,
    tools/compiler/ddr_image.hpp) over device memory; ctx=False keeps the
    bookkeeping only (no device memory)."""

    PAGE = 4096

    def __init__(self, capacity: int, ctx: Context | None | bool = None):
        if ctx is False:
            handle_ctx = None
        else:
            handle_ctx = (ctx or default_context()).handle
        h = C.c_void_p()
        _check(lib().hb_image_create(handle_ctx, capacity, C.byref(h)))
        self.handle = h

    def close(self) -> None:
        if self.handle:
            lib().hb_image_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def alloc(self, name: str, size: int, align: int = 0) -> int:
        off = C.c_uint64()
        _check(lib().hb_image_alloc(self.handle, name.encode(), size, align, C.byref(off)))
        return off.value

    def set_reuse(self, reuse: bool) -> None:
        lib().hb_image_set_reuse(self.handle, 1 if reuse else 0)

    def define(self, name: str, offset: int, size: int) -> None:
        _check(lib().hb_image_define(self.handle, name.encode(), offset, size))

    def put(self, offset: int, data: bytes) -> None:
        buf = C.create_string_buffer(bytes(data), len(data))
        _check(lib().hb_image_put(self.handle, offset, buf, len(data)))

    def get(self, offset: int, size: int) -> bytes:
        buf = C.create_string_buffer(size)
        _check(lib().hb_image_get(self.handle, offset, buf, size))
        return buf.raw

    def region(self, name: str) -> tuple[int, int]:
        off, size = C.c_uint64(), C.c_uint64()
        _check(lib().hb_image_region(self.handle, name.encode(), C.byref(off), C.byref(size)))
        return off.value, size.value

    def regions(self) -> list[tuple[str, int, int]]:
        out = []
        for i in range(int(lib().hb_image_region_count(self.handle))):
            name, off, size = C.c_char_p(), C.c_uint64(), C.c_uint64()
            _check(lib().hb_image_region_at(self.handle, i, C.byref(name), C.byref(off),
                                            C.byref(size)))
            out.append((name.value.decode(), off.value, size.value))
        return out

    def end(self) -> int:
        return int(lib().hb_image_end(self.handle))

    def ptr(self, name: str) -> int:
        """Device address of a region."""
        base = lib().hb_image_base(self.handle)
        if not base:
            raise HbError(HB_EINVAL, "the image has no device memory")
        return int(base) + self.region(name)[0]


def split8(src, rows: int, row_words: int, hi, lo, src_stride: int | None = None,
           ctx: Context | None = None, sync: bool = True) -> None:
    """SPLIT8 (dma_engine.cpp:303-333) on device DDR words: MXINT8 rows ->
    the W8 planes hi, lo ([rows/2][row_words] x 144 B each) of the matrix
    whose columns are the tokens."""
    ctx = ctx or default_context()
    stride = row_words * 144 if src_stride is None else src_stride
    fn = lib().hb_split8 if sync else lib().hb_split8_async
    _check(fn(ctx.handle, _ptr(src), stride, rows, row_words, _ptr(hi), _ptr(lo)))


def t32_split8(src, rows: int, row_words: int, hi, lo, src_stride: int | None = None,
               ctx: Context | None = None, sync: bool = True) -> None:
    """T32_SPLIT8 (dma_engine.cpp:336-398): the W8 planes of the transpose,
    with per-block scale alignment ([4*row_words][rows/8] x 144 B each)."""
    ctx = ctx or default_context()
    stride = row_words * 144 if src_stride is None else src_stride
    fn = lib().hb_t32_split8 if sync else lib().hb_t32_split8_async
    _check(fn(ctx.handle, _ptr(src), stride, rows, row_words, _ptr(hi), _ptr(lo)))


def encode_mxint8(x, rows: int, cols: int, out, ctx: Context | None = None) -> None:
    """EncodeMxint8 + PackAbuf of a device fp32 [rows][cols] into DDR words."""
    ctx = ctx or default_context()
    _check(lib().hb_encode_mxint8(ctx.handle, _ptr(x), rows, cols, _ptr(out)))


def encode_mxfp8(x, rows: int, cols: int, out, ctx: Context | None = None) -> None:
    """hb_encode_mxfp8: a device fp32 [rows][cols] as MXFP8 E4M3 DDR words."""
    ctx = ctx or default_context()
    _check(lib().hb_encode_mxfp8(ctx.handle, _ptr(x), rows, cols, _ptr(out)))


# ---------------------------------------------------- serving operators --
# These take torch tensors: sizes, types and strides come from them.  Without
# `ctx` a call is ordered on torch's current stream, like torch's own; with one
# it is ordered on that context's stream (Context.set_stream), and with sync
# False the caller orders torch's work on the same tensors with it.  Steps of
# few tokens wait for the host, so the descriptors are packed in one go, and
# the checks read each property of a tensor once.

HB_TYPE_F32, HB_TYPE_BF16, HB_TYPE_F16 = range(3)
#: the descriptors of include/hotarubi_gpu.h, field for field
KV_PLAN_DESC = struct.Struct("@10P6I")
NORM_ROPE_DESC = struct.Struct("@4P8Q3PQPf8I3I")
KV_ROWS_DESC = struct.Struct("@P4I2P4QP2I")
KV_ATTENTION_DESC = struct.Struct("@P4I2P4Q4P9I2f")
KV8_ATTENTION_DESC = struct.Struct("@P4I2P4Q4P10I2f")
KV_FORK_DESC = struct.Struct("@9P6I")
KV_COPY_DESC = struct.Struct("@2P2Q3I")
KV_FREE_DESC = struct.Struct("@7P7I")
KV_COMPACT_DESC = struct.Struct("@7P8I")
LOGPROBS_DESC = struct.Struct("@PQ5P4If")
_types = None  # (torch.dtype -> hb_type, int32, uint8, float64, float32)


def _torch_types():
    global _types
    import torch
    _types = ({torch.float32: HB_TYPE_F32, torch.bfloat16: HB_TYPE_BF16,
               torch.float16: HB_TYPE_F16}, torch.int32, torch.uint8, torch.float64,
              torch.float32)
    return _types


def _invalid(message: str):
    return HbError(HB_EINVAL, message)


_own = threading.local()  # a host thread's contexts, by device and stream


def _torch_context(t, name: str) -> Context:
    """The context of a call that names none: one of its own for torch's
    current stream on t's device, so that the call comes after the torch work
    issued before it and before what is issued next, and calls on two streams
    do not share a workspace."""
    import torch
    device = t.get_device()
    if device < 0:
        raise _invalid(f"{name} is on {t.device}, not on a GPU")
    stream = torch.cuda.current_stream(device).cuda_stream
    contexts = _own.__dict__
    ctx = contexts.get((device, stream))
    if ctx is None:
        ctx = Context(device)
        ctx.set_stream(stream)
        contexts[device, stream] = ctx
    return ctx


def _vector(t, dtype, name: str, count: int, device: int) -> int:
    """Address of a contiguous vector of `count` elements (-1: any)."""
    if t.dtype is not dtype or t.stride() != (1,) or t.get_device() != device or \
            (t.shape[0] != count and count >= 0):
        if t.dtype is not dtype or t.dim() != 1 or not t.is_contiguous() or \
                (t.shape[0] != count and count >= 0):
            raise _invalid(f"{name} must be {'n' if count < 0 else count} contiguous {dtype} "
                           f"elements, not {tuple(t.shape)} of {t.dtype}")
        _place(t, name, device)
    return t.data_ptr()


def _place(t, name: str, device: int) -> None:
    if t.get_device() != device:
        raise _invalid(f"{name} is on {t.device}, the context on cuda:{device}")


def _heads(t, dtype, name: str, shape, device: int):
    """(address, token stride, head stride) of [tokens][heads][dim] rows."""
    stride = t.stride()
    if t.dtype is not dtype or len(stride) != 3 or (shape is not None and t.shape != shape):
        raise _invalid(f"{name} is {tuple(t.shape)} of {t.dtype}, not "
                       f"{'[tokens][heads][dim]' if shape is None else tuple(shape)} of {dtype}")
    if stride[2] != 1 and t.shape[2] > 1 and t.numel() > 0:
        raise _invalid(f"{name}: a head's elements must be neighbours")
    if t.get_device() != device:
        _place(t, name, device)
    return t.data_ptr(), stride[0], stride[1]


def _table(t, i32, device: int, name: str = "table"):
    """(address, rows, entries of a row, row stride) of a block table."""
    stride = t.stride()
    if t.dtype is not i32 or len(stride) != 2 or \
            (stride[1] != 1 and t.shape[1] > 1 and t.numel() > 0):
        raise _invalid(f"{name} must be int32 rows, not {tuple(t.shape)} of {t.dtype}")
    if t.get_device() != device:
        _place(t, name, device)
    batch, columns = t.shape
    return t.data_ptr(), batch, columns, stride[0]


def _cache(t, u8, device: int):
    """(address, pages, heads, page size, head size) of a cache."""
    size = t.shape
    if t.dtype is not u8 or len(size) != 4 or size[3] % 34 or not t.is_contiguous():
        raise _invalid("the cache must be contiguous uint8 [pages][heads][page / 32][34 dim], not "
                       f"{tuple(size)} of {t.dtype}")
    if t.get_device() != device:
        _place(t, "cache", device)
    return t.data_ptr(), size[0], size[1], 32 * size[2], size[3] // 34


def _cache8(t, u8, device: int):
    """The same of a cache of 8 bits."""
    size = t.shape
    if t.dtype is not u8 or len(size) != 4 or size[3] % 64 != 16 or not t.is_contiguous():
        raise _invalid("the cache must be contiguous uint8 [pages][heads][page / 32][64 dim + 16], "
                       f"not {tuple(size)} of {t.dtype}")
    if t.get_device() != device:
        _place(t, "cache", device)
    return t.data_ptr(), size[0], size[1], 32 * size[2], size[3] // 64


def _pairs(t, i32, device: int) -> int:
    """Address of [count][2] page numbers."""
    if t.dtype is not i32 or t.dim() != 2 or t.shape[1] != 2 or not t.is_contiguous():
        raise _invalid(f"pairs must be contiguous int32 [n][2], not {tuple(t.shape)} of {t.dtype}")
    _place(t, "pairs", device)
    return t.data_ptr()


def _kind(kinds, t, name: str) -> int:
    kind = kinds.get(t.dtype)
    if kind is None:
        raise _invalid(f"{name} is {t.dtype} (float32, bfloat16 or float16)")
    return kind


def _desc(layout: struct.Struct, *values) -> bytes:
    try:
        return layout.pack(*values)
    except struct.error as e:  # a size that its field does not hold
        raise _invalid(f"argument out of range: {e}") from None


def kv_plan(lens, new_tokens, free_pages, free_count, table, page_size: int, cu, kv_lens, slots,
            positions, status, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_plan: a serving step's plan on the device.  lens, new_tokens int32
    [batch]; free_pages int32 (a stack of free_count [1] pages); table int32
    [batch][columns] gets the new pages; cu [batch + 1], kv_lens [batch], slots
    and positions [size], status [2] (pages taken, requests refused) are
    written."""
    ctx = ctx or _torch_context(lens, "lens")
    i32, dev = (_types or _torch_types())[1], ctx.device
    at, batch, columns, stride = _table(table, i32, dev)
    slots_at = _vector(slots, i32, "slots", -1, dev)
    free_at = _vector(free_pages, i32, "free_pages", -1, dev)
    size = slots.shape[0]
    d = _desc(KV_PLAN_DESC, _vector(lens, i32, "lens", batch, dev),
              _vector(new_tokens, i32, "new_tokens", batch, dev), free_at,
              _vector(free_count, i32, "free_count", 1, dev), at,
              _vector(cu, i32, "cu", batch + 1, dev),
              _vector(kv_lens, i32, "kv_lens", batch, dev), slots_at,
              _vector(positions, i32, "positions", size, dev),
              _vector(status, i32, "status", 2, dev), batch, columns, stride, page_size, size,
              free_pages.shape[0])
    _check((lib().hb_kv_plan if sync else lib().hb_kv_plan_async)(ctx.handle, d))


def norm_rope(q, positions, inv_freq, q_out, k=None, k_out=None, gamma_q=None, gamma_k=None,
              eps: float = 1e-6, sections=None, interleaved: bool = False,
              ctx: Context | None = None, sync: bool = True) -> None:
    """hb_norm_rope: RMS norm of every head of q (and k) with gamma (None: not
    normalised) and the rotation of its first 2 * len(inv_freq) elements.  q
    [tokens][heads][dim]; positions int32 [axes][tokens] (or [tokens]);
    inv_freq float64; sections: the pairs of each axis."""
    ctx = ctx or _torch_context(q, "q")
    kinds, i32, _, f64, f32 = _types or _torch_types()
    kind, dev, dtype = _kind(kinds, q, "q"), ctx.device, q.dtype
    qa, qt, qh = _heads(q, dtype, "q", None, dev)
    tokens, heads, dim = q.shape
    oa, ot, oh = _heads(q_out, dtype, "q_out", q.shape, dev)
    ka = kt = kh = pa = pt = ph = k_heads = 0
    if k is not None:
        if k_out is None:
            raise _invalid("k without k_out")
        ka, kt, kh = _heads(k, dtype, "k", None, dev)
        k_tokens, k_heads, k_dim = k.shape
        if k_tokens != tokens or k_dim != dim:
            raise _invalid(f"k is {tuple(k.shape)}, q {tuple(q.shape)}")
        pa, pt, ph = _heads(k_out, dtype, "k_out", k.shape, dev)
    if positions.dim() == 1:
        positions = positions[None]
    stride = positions.stride()
    if positions.dtype is not i32 or len(stride) != 2 or positions.shape[1] != tokens or \
            (tokens > 1 and stride[1] != 1):
        raise _invalid(f"positions must be int32 [axes][{tokens}], not "
                       f"{tuple(positions.shape)} of {positions.dtype}")
    if positions.get_device() != dev:
        _place(positions, "positions", dev)
    axes = positions.shape[0]
    freq = _vector(inv_freq, f64, "inv_freq", -1, dev)
    half = inv_freq.shape[0]
    if sections is None:
        sections = (half,)
    if len(sections) != axes or not 1 <= axes <= 3:
        raise _invalid(f"sections {tuple(sections)} for {axes} position axes")
    d = _desc(NORM_ROPE_DESC, qa, ka, oa, pa, qt, qh, kt, kh, ot, oh, pt, ph,
              0 if gamma_q is None else _vector(gamma_q, f32, "gamma_q", dim, dev),
              0 if gamma_k is None else _vector(gamma_k, f32, "gamma_k", dim, dev),
              positions.data_ptr(), stride[0], freq, eps, kind, tokens, heads, k_heads, dim,
              2 * half, 1 if interleaved else 0, axes, *sections, *(0,) * (3 - axes))
    _check((lib().hb_norm_rope if sync else lib().hb_norm_rope_async)(ctx.handle, d))


def _kv_rows(fn, k, v, slots, cache, ctx, layout=_cache) -> None:
    kinds, i32, u8, _, _ = _types or _torch_types()
    dev, dtype = ctx.device, k.dtype
    c = layout(cache, u8, dev)
    kind = _kind(kinds, k, "k")
    ka, kt, kh = _heads(k, dtype, "k", None, dev)
    tokens, heads, dim = k.shape
    if heads != c[2] or dim != c[4]:
        raise _invalid(f"k is {tuple(k.shape)}, the cache has {c[2]} heads of {c[4]}")
    va, vt, vh = _heads(v, dtype, "v", k.shape, dev)
    _check(fn(ctx.handle, _desc(KV_ROWS_DESC, *c, ka, va, kt, kh, vt, vh,
                                _vector(slots, i32, "slots", tokens, dev), kind, tokens)))


def kv_cache_shape(pages: int, heads: int, page_size: int, dim: int) -> tuple[int, int, int, int]:
    """Shape of a paged MXFP4 cache (uint8)."""
    return pages, heads, page_size // 32, 34 * dim


def kv_append(k, v, slots, cache, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_append: rows k, v [tokens][heads][dim] into the cache (uint8
    [pages][heads][page / 32][34 dim]) at int32 slots."""
    _kv_rows(lib().hb_kv_append if sync else lib().hb_kv_append_async, k, v, slots, cache,
             ctx or _torch_context(k, "k"))


def kv_read(k, v, slots, cache, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_read: the stored values of slots into k, v [tokens][heads][dim]."""
    _kv_rows(lib().hb_kv_read if sync else lib().hb_kv_read_async, k, v, slots, cache,
             ctx or _torch_context(k, "k"))


def _attention_desc(dev: int, q, out, cache, table, cu, kv_lens, max_new, max_kv, scale, prefix,
                    window, softcap, sinks=()) -> bytes:
    kinds, i32, u8, _, _ = _types or _torch_types()
    dtype = q.dtype
    layout, c = (KV8_ATTENTION_DESC, _cache8(cache, u8, dev)) if sinks else \
        (KV_ATTENTION_DESC, _cache(cache, u8, dev))
    kind = _kind(kinds, q, "q")
    qa, qt, qh = _heads(q, dtype, "q", None, dev)
    tokens, heads, dim = q.shape
    if dim != c[4]:
        raise _invalid(f"q has heads of {dim} elements, the cache of {c[4]}")
    oa, ot, oh = _heads(out, dtype, "out", q.shape, dev)
    at, batch, columns, stride = _table(table, i32, dev)
    return _desc(layout, *c, qa, oa, qt, qh, ot, oh, at,
                 _vector(cu, i32, "cu", batch + 1, dev),
                 _vector(kv_lens, i32, "kv_lens", batch, dev),
                 0 if prefix is None else _vector(prefix, i32, "prefix", batch, dev), kind, tokens,
                 heads, batch, columns, stride, max_new, max_kv, window, *sinks, scale, softcap)


def kv_attention(q, out, cache, table, cu, kv_lens, max_new: int, max_kv: int, scale: float,
                 prefix=None, window: int = 0, softcap: float = 0.0,
                 ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_attention: q [tokens][heads][dim] of ragged requests (rows
    [cu[b], cu[b + 1]) are the last tokens of request b's kv_lens[b]) against
    the paged cache, into out.  Causal; prefix int32 [batch]: leading keys that
    every row sees; window: keys a row sees, itself among them (0: all);
    softcap: scores as softcap * tanh(score / softcap)."""
    ctx = ctx or _torch_context(q, "q")
    d = _attention_desc(ctx.device, q, out, cache, table, cu, kv_lens, max_new, max_kv, scale,
                        prefix, window, softcap)
    _check((lib().hb_kv_attention if sync else lib().hb_kv_attention_async)(ctx.handle, d))


#: hb_kv_way's `way`
KV_WAYS = ("none", "rows", "splits", "shares", "prompt")
KV_WAY = struct.Struct("@4IQ")


def kv_attention_way(q, out, cache, table, cu, kv_lens, max_new: int, max_kv: int, scale: float,
                     prefix=None, window: int = 0, softcap: float = 0.0):
    """hb_kv_attention_way: how kv_attention would divide this call's work on
    the current device: (one of KV_WAYS, 16-row tiles of a wave, splits of the
    keys, bytes of workspace).  Nothing is run."""
    way = C.create_string_buffer(KV_WAY.size)
    _check(lib().hb_kv_attention_way(
        _attention_desc(q.get_device(), q, out, cache, table, cu, kv_lens, max_new, max_kv, scale,
                        prefix, window, softcap), way))
    kind, tiles, splits, _, workspace = KV_WAY.unpack(way.raw)
    return KV_WAYS[kind], tiles, splits, workspace


def kv8_cache_shape(pages: int, heads: int, page_size: int, dim: int) -> tuple[int, int, int, int]:
    """Shape of a paged cache of 8 bits (uint8); it starts as zeros."""
    return pages, heads, page_size // 32, 64 * dim + 16


def kv8_append(k, v, slots, cache, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv8_append: rows k, v [tokens][heads][dim] into the cache (uint8
    [pages][heads][page / 32][64 dim + 16]) at int32 slots, the tokens of a
    block of 32 in their order."""
    _kv_rows(lib().hb_kv8_append if sync else lib().hb_kv8_append_async, k, v, slots, cache,
             ctx or _torch_context(k, "k"), _cache8)


def kv8_read(k, v, slots, cache, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv8_read: the stored values of slots into k, v [tokens][heads][dim]."""
    _kv_rows(lib().hb_kv8_read if sync else lib().hb_kv8_read_async, k, v, slots, cache,
             ctx or _torch_context(k, "k"), _cache8)


def kv8_attention(q, out, cache, table, cu, kv_lens, max_new: int, max_kv: int, scale: float,
                  prefix=None, window: int = 0, sinks: int = 0, softcap: float = 0.0,
                  ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv8_attention: kv_attention over a cache of 8 bits.  sinks: with a
    window, the first tokens that stay visible to the rows behind them."""
    ctx = ctx or _torch_context(q, "q")
    d = _attention_desc(ctx.device, q, out, cache, table, cu, kv_lens, max_new, max_kv, scale,
                        prefix, window, softcap, (sinks,))
    _check((lib().hb_kv8_attention if sync else lib().hb_kv8_attention_async)(ctx.handle, d))


def kv8_attention_way(q, out, cache, table, cu, kv_lens, max_new: int, max_kv: int, scale: float,
                      prefix=None, window: int = 0, sinks: int = 0, softcap: float = 0.0):
    """hb_kv8_attention_way: kv_attention_way for kv8_attention."""
    way = C.create_string_buffer(KV_WAY.size)
    _check(lib().hb_kv8_attention_way(
        _attention_desc(q.get_device(), q, out, cache, table, cu, kv_lens, max_new, max_kv, scale,
                        prefix, window, softcap, (sinks,)), way))
    kind, tiles, splits, _, workspace = KV_WAY.unpack(way.raw)
    return KV_WAYS[kind], tiles, splits, workspace


def kv_fork(table, lens, source, target, free_pages, free_count, page_size: int, lens_out, pairs,
            status, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_fork: request target[i] goes on from request source[i]'s tokens.
    table int32 [batch][columns] gets the targets' entries; lens int32 [batch];
    source, target int32 [forks]; free_pages int32 (a stack of free_count [1]
    pages); lens_out [batch], pairs [forks][2] (for kv_copy) and status [2]
    (pages taken, forks refused) are written."""
    ctx = ctx or _torch_context(table, "table")
    i32, dev = (_types or _torch_types())[1], ctx.device
    at, batch, columns, stride = _table(table, i32, dev)
    source_at = _vector(source, i32, "source", -1, dev)
    forks = source.shape[0]
    pairs_at = _pairs(pairs, i32, dev)
    if pairs.shape[0] != forks:
        raise _invalid(f"{pairs.shape[0]} pairs for {forks} forks")
    free_at = _vector(free_pages, i32, "free_pages", -1, dev)
    d = _desc(KV_FORK_DESC, at, _vector(lens, i32, "lens", batch, dev), source_at,
              _vector(target, i32, "target", forks, dev), free_at,
              _vector(free_count, i32, "free_count", 1, dev),
              _vector(lens_out, i32, "lens_out", batch, dev), pairs_at,
              _vector(status, i32, "status", 2, dev), batch, columns, stride, page_size, forks,
              free_pages.shape[0])
    _check((lib().hb_kv_fork if sync else lib().hb_kv_fork_async)(ctx.handle, d))


def kv_copy(cache, pairs, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_copy: page pairs[i][0] over page pairs[i][1] (int32 [n][2]) of a
    cache, of 4 or 8 bits: uint8 [pages][heads][page / 32][record], or with
    [layers] in front of that."""
    ctx = ctx or _torch_context(cache, "cache")
    _, i32, u8, _, _ = _types or _torch_types()
    size = cache.shape
    if cache.dtype is not u8 or len(size) not in (4, 5) or not cache.is_contiguous():
        raise _invalid("the cache must be contiguous uint8 [layers][pages][heads][page / 32]"
                       f"[record], not {tuple(size)} of {cache.dtype}")
    _place(cache, "cache", ctx.device)
    page = size[-3] * size[-2] * size[-1]
    d = _desc(KV_COPY_DESC, cache.data_ptr(), _pairs(pairs, i32, ctx.device), page,
              page * size[-4], size[-4], size[0] if len(size) == 5 else 1, pairs.shape[0])
    _check((lib().hb_kv_copy if sync else lib().hb_kv_copy_async)(ctx.handle, d))


def kv_free(table, lens, rows, pages: int, free_pages, free_count, page_size: int, lens_out,
            status, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_free: requests `rows` (int32) end: their pages that no other
    request names go on the stack free_pages above its free_count [1] pages.
    pages: of the cache; lens_out [batch] (0 for them) and status [2] (pages
    put back, pages without room) are written."""
    ctx = ctx or _torch_context(table, "table")
    i32, dev = (_types or _torch_types())[1], ctx.device
    at, batch, columns, stride = _table(table, i32, dev)
    d = _desc(KV_FREE_DESC, at, _vector(lens, i32, "lens", batch, dev),
              _vector(rows, i32, "rows", -1, dev), _vector(free_pages, i32, "free_pages", -1, dev),
              _vector(free_count, i32, "free_count", 1, dev),
              _vector(lens_out, i32, "lens_out", batch, dev),
              _vector(status, i32, "status", 2, dev), batch, columns, stride, page_size,
              rows.shape[0], pages, free_pages.shape[0])
    _check((lib().hb_kv_free if sync else lib().hb_kv_free_async)(ctx.handle, d))


def kv_compact(table, lens, pages: int, page_size: int, table_out, free_pages, free_count, pairs,
               status, ctx: Context | None = None, sync: bool = True) -> None:
    """hb_kv_compact: renumbers a cache of `pages` pages so that those in use
    are the first.  table_out [batch][columns] (may be table), free_pages (at
    least `pages`), free_count [1], pairs [at least pages / 2][2] (for kv_copy)
    and status [2] (pages in use, pages that move) are written."""
    ctx = ctx or _torch_context(table, "table")
    i32, dev = (_types or _torch_types())[1], ctx.device
    at, batch, columns, stride = _table(table, i32, dev)
    out_at, out_batch, out_columns, out_stride = _table(table_out, i32, dev, "table_out")
    if (out_batch, out_columns) != (batch, columns):
        raise _invalid(f"table_out is {tuple(table_out.shape)}, table {tuple(table.shape)}")
    d = _desc(KV_COMPACT_DESC, at, _vector(lens, i32, "lens", batch, dev), out_at,
              _vector(free_pages, i32, "free_pages", -1, dev),
              _vector(free_count, i32, "free_count", 1, dev), _pairs(pairs, i32, dev),
              _vector(status, i32, "status", 2, dev), batch, columns, stride, out_stride,
              page_size, pages, free_pages.shape[0], pairs.shape[0])
    _check((lib().hb_kv_compact if sync else lib().hb_kv_compact_async)(ctx.handle, d))


def _row_list(t, dtype, name: str, rows: int, top: int, device: int) -> int:
    """Address of contiguous [rows][top]."""
    if t.dtype is not dtype or tuple(t.shape) != (rows, top) or not t.is_contiguous():
        raise _invalid(f"{name} must be contiguous {dtype} [{rows}][{top}], not "
                       f"{tuple(t.shape)} of {t.dtype}")
    _place(t, name, device)
    return t.data_ptr()


def token_logprobs(logits, tokens=None, logprobs=None, entropy=None, top_ids=None,
                   top_logprobs=None, scale: float = 1.0, ctx: Context | None = None,
                   sync: bool = True) -> None:
    """hb_token_logprobs: of each row of scale * logits [rows][vocab], the log
    probability of tokens[row] (int32; below 0: none) into logprobs, the
    entropy, and the most likely tokens' columns and log probabilities into
    top_ids (int32) and top_logprobs [rows][top].  Results are fp32; what is
    None is left out."""
    ctx = ctx or _torch_context(logits, "logits")
    kinds, i32, _, _, f32 = _types or _torch_types()
    kind, dev = _kind(kinds, logits, "logits"), ctx.device
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise _invalid(f"logits must be rows of neighbouring elements, not {tuple(logits.shape)} "
                       f"with strides {logits.stride()}")
    _place(logits, "logits", dev)
    rows, vocab = logits.shape
    if (tokens is None) != (logprobs is None) or (top_ids is None) != (top_logprobs is None):
        raise _invalid("tokens and logprobs, top_ids and top_logprobs go together")
    top = ids_at = top_at = 0
    if top_ids is not None:
        if top_ids.dim() != 2 or top_ids.shape[1] < 1:
            raise _invalid(f"top_ids is {tuple(top_ids.shape)}, not [rows][top]")
        top = top_ids.shape[1]
        ids_at = _row_list(top_ids, i32, "top_ids", rows, top, dev)
        top_at = _row_list(top_logprobs, f32, "top_logprobs", rows, top, dev)
    d = _desc(LOGPROBS_DESC, logits.data_ptr(), logits.stride(0),
              0 if tokens is None else _vector(tokens, i32, "tokens", rows, dev),
              0 if logprobs is None else _vector(logprobs, f32, "logprobs", rows, dev),
              0 if entropy is None else _vector(entropy, f32, "entropy", rows, dev), ids_at,
              top_at, kind, rows, vocab, top, scale)
    _check((lib().hb_token_logprobs if sync else lib().hb_token_logprobs_async)(ctx.handle, d))
