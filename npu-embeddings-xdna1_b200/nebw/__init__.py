"""Python front of libnebw (include/nebw.h) through ctypes.

This module is plumbing for tests, the benchmark and Python callers: the
product is the C ABI and the CUDA kernels behind it.  There is no CPU path
here: if libnebw.so is missing or no sm_100 GPU is present, the calls fail
by name.

Device buffers may be torch CUDA tensors (their data_ptr is passed) or raw
integer device addresses.
"""

from __future__ import annotations

import ctypes as C
import os
import re
from pathlib import Path

import numpy as np

PKG_DIR = Path(__file__).resolve().parent.parent          # npu-embeddings-xdna1_b200/
REPO_DIR = PKG_DIR.parent
LIB_PATH = Path(os.environ["NEBW_LIB"]) if os.environ.get("NEBW_LIB") else PKG_DIR / "libnebw.so"
HEADER_PATH = REPO_DIR / "include" / "nebw.h"

ABI = (5, 1)  # NEBW_ABI_VERSION and _REVISION of include/nebw.h
F32, BF16 = 0, 1
ACT_NONE, ACT_GELU8, ACT_GELU_ERF = 0, 1, 2
GATE_SILU, GATE_GELU_ERF = 0, 1
POOL_MEAN, POOL_CLS = 0, 1
ROPE_HALF, ROPE_PAIRS = 0, 1
HEADNORM_NONE, HEADNORM_RMS, HEADNORM_LAYER = 0, 1, 2
ROUTE_SOFTMAX, ROUTE_SIGMOID = 0, 1
MAX_TOP_K = 16  # experts of a row


class NebwError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"nebw error {code}: {msg}")
        self.code = code


class Config(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "num_layers", "hidden", "num_heads", "head_dim", "intermediate", "vocab_size",
        "max_seq_len", "type_vocab_size", "pooling", "l2_normalize", "activation")] + [
        ("layer_norm_eps", C.c_float)] + [(n, C.c_int32) for n in (
        "gated_ffn", "gated_act", "rope", "reserved0")] + [("rope_theta", C.c_double)]


class VitConfig(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "num_layers", "hidden", "num_heads", "head_dim", "intermediate", "image_size",
        "patch_size", "num_channels")] + [("layer_norm_eps", C.c_float)]


class RopeScaling(C.Structure):
    _fields_ = [("kind", C.c_int32), ("reserved0", C.c_int32), ("orig_len", C.c_int64),
                ("factor", C.c_double), ("fast", C.c_double), ("slow", C.c_double),
                ("attn_scale", C.c_double)]


class Heads(C.Structure):
    """The query or key heads of packed rows (nebw_heads)."""

    _fields_ = [("x", C.c_void_p), ("out", C.c_void_p), ("stride", C.c_int64),
                ("out_stride", C.c_int64), ("heads", C.c_int32), ("reserved0", C.c_int32),
                ("gamma", C.c_void_p), ("beta", C.c_void_p)]

    @classmethod
    def of(cls, x, heads: int, out=None, gamma=None, beta=None):
        """Heads of a 2-D torch CUDA tensor [rows, heads * head_dim] (a column
        slice of Q|K|V rows, say), in place or into `out` of the same shape.
        The object keeps the tensors alive."""
        out = x if out is None else out
        for t in (x, out):
            if t.dim() != 2 or t.stride(1) != 1 or t.shape[1] % heads:
                raise ValueError("heads are rows of a 2-D tensor with adjacent elements")
        if out.shape != x.shape or out.dtype != x.dtype:
            raise ValueError("the heads' output must have their shape and dtype")
        for t in (gamma, beta):
            if t is not None and (str(t.dtype) != "torch.float32" or not t.is_contiguous()
                                  or t.numel() != x.shape[1] // heads):
                raise ValueError("a head norm's weights are head_dim contiguous fp32 values")
        h = cls(x.data_ptr(), out.data_ptr(), x.stride(0), out.stride(0), heads, 0, _addr(gamma),
                _addr(beta))
        h.dtype = _dtype(x)
        h.tensors = tuple(t for t in (x, out, gamma, beta) if t is not None)
        h.rows, h.head_dim = x.shape[0], x.shape[1] // heads
        gpus = {t.get_device() for t in h.tensors}
        h.gpu = gpus.pop() if len(gpus) == 1 else -1  # -1: not on one GPU
        return h


_lib = None


def header_functions() -> list[str]:
    """Names of every function include/nebw.h declares."""
    text = HEADER_PATH.read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    return sorted(set(re.findall(r"\b(nebw_[a-z0-9_]+)\s*\(", text)))


def lib() -> C.CDLL:
    """Load libnebw.so (once).  Raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise FileNotFoundError(
            f"{LIB_PATH} is not built; run `python __graft_entry__.py build` (or build()) first")
    L = C.CDLL(str(LIB_PATH))
    # a library of an earlier build is refused here, not at some later call
    got = (L.nebw_abi_version(), L.nebw_abi_revision() if hasattr(L, "nebw_abi_revision") else 0)
    if got[0] != ABI[0] or got[1] < ABI[1]:
        raise NebwError(1, f"{LIB_PATH} is of another build: ABI {got[0]}.{got[1]}, and "
                           f"{ABI[0]}.{ABI[1]} is required; run build() again")
    vp, i64, i32 = C.c_void_p, C.c_int64, C.c_int32
    sig = {
        "nebw_last_error": ([], C.c_char_p),
        "nebw_abi_version": ([], C.c_int),
        "nebw_abi_revision": ([], C.c_int),
        "nebw_open": ([C.c_int, C.POINTER(vp)], C.c_int),
        "nebw_close": ([vp], C.c_int),
        "nebw_sync": ([vp], C.c_int),
        "nebw_alloc": ([vp, C.c_size_t, C.POINTER(vp)], C.c_int),
        "nebw_free": ([vp, vp], C.c_int),
        "nebw_copy_h2d": ([vp, vp, vp, C.c_size_t], C.c_int),
        "nebw_copy_d2h": ([vp, vp, vp, C.c_size_t], C.c_int),
        "nebw_device_info": ([vp, C.POINTER(C.c_int), C.POINTER(C.c_int), C.POINTER(C.c_int)], C.c_int),
        "nebw_stage_weight": ([vp, vp, C.c_int, i64, i64, C.POINTER(C.c_uint64)], C.c_int),
        "nebw_release_weight": ([vp, C.c_uint64], C.c_int),
        "nebw_gemm": ([vp, C.c_uint64, vp, i64, i64, i64, vp, vp, C.c_int, vp, C.c_int, vp], C.c_int),
        "nebw_layernorm": ([vp, vp, vp, C.c_int, vp, vp, C.c_float, i64, i64, vp, vp], C.c_int),
        "nebw_attention": ([vp, vp, i64, vp, vp, i32, i32, i32, i32, vp, vp], C.c_int),
        "nebw_pack_offsets": ([vp, vp, i32, i32, vp, vp, vp], C.c_int),
        "nebw_embed_ln": ([vp, vp, vp, vp, i32, i32, vp, i32, vp, vp, vp, vp, C.c_float, i32, vp,
                           vp, vp], C.c_int),
        "nebw_pool_l2": ([vp, vp, vp, vp, i32, i32, C.c_int, C.c_int, vp, vp], C.c_int),
        "nebw_narrow_bf16": ([vp, vp, i64, vp, vp], C.c_int),
        "nebw_model_create": ([vp, C.POINTER(Config), C.POINTER(vp)], C.c_int),
        "nebw_model_set_rope_freq": ([vp, C.POINTER(C.c_double), C.c_int32], C.c_int),
        "nebw_model_set_tensor": ([vp, C.c_char_p, vp, C.c_int, i64, i64], C.c_int),
        "nebw_model_load_npue": ([vp, C.c_char_p, C.POINTER(vp)], C.c_int),
        "nebw_tma_layout_hash": ([], C.c_char_p),
        "nebw_npue_gemm_kn": ([C.c_char_p, C.c_char_p, vp, i64, i64], C.c_int),
        "nebw_model_set_gemm_nk": ([vp, C.c_char_p, vp, i64, i64], C.c_int),
        "nebw_model_destroy": ([vp], C.c_int),
        "nebw_model_get_config": ([vp, C.POINTER(Config)], C.c_int),
        "nebw_encode": ([vp, vp, vp, i32, i32, vp], C.c_int),
        "nebw_encode_device": ([vp, vp, vp, i32, i32, vp, vp], C.c_int),
        "nebw_encode_launch_count": ([vp, i32], C.c_int),
        "nebw_encode_device_static": ([vp, vp, vp, i32, i32, vp, vp], C.c_int),
        "nebw_set_attention_kernel": ([vp, C.c_int], C.c_int),
        "nebw_model_profile": ([vp, C.c_int], C.c_int),
        "nebw_model_profile_collect": ([vp, C.POINTER(C.c_int64), C.POINTER(C.c_double)], C.c_int),
        "nebw_vit_create": ([vp, C.POINTER(VitConfig), C.POINTER(vp)], C.c_int),
        "nebw_vit_set_tensor": ([vp, C.c_char_p, vp, C.c_int, i64, i64], C.c_int),
        "nebw_vit_load_npue": ([vp, C.c_char_p, C.POINTER(vp)], C.c_int),
        "nebw_vit_get_config": ([vp, C.POINTER(VitConfig)], C.c_int),
        "nebw_vit_destroy": ([vp], C.c_int),
        "nebw_vit_encode_device": ([vp, vp, i32, vp, vp], C.c_int),
        "nebw_vit_encode": ([vp, vp, i32, vp], C.c_int),
        "nebw_vit_launch_count": ([vp], C.c_int),
        "nebw_vit_profile": ([vp, C.c_int], C.c_int),
        "nebw_vit_profile_collect": ([vp, C.POINTER(C.c_int64), C.POINTER(C.c_double)], C.c_int),
        "nebw_check_bounded_wait": ([vp, i64, C.POINTER(i32)], C.c_int),
        "nebw_quantise_rows": ([vp, vp, i64, i64, vp, vp, vp, vp], C.c_int),
        "nebw_stage_weight_i8": ([vp, vp, i64, i64, C.POINTER(C.c_uint64)], C.c_int),
        "nebw_gemm_i8": ([vp, C.c_uint64, vp, vp, i64, i64, i64, vp, vp, C.c_int, vp, vp], C.c_int),
        "nebw_gemm_i8_ex": ([vp, C.c_uint64, vp, vp, i64, i64, i64, vp, vp, C.c_int, vp, C.c_int,
                             vp], C.c_int),
        "nebw_quantise_rows_bf16": ([vp, vp, i64, i64, vp, vp, vp, vp], C.c_int),
        "nebw_layernorm_quant": ([vp, vp, vp, vp, vp, C.c_float, i64, i64, vp, vp, vp, vp],
                                 C.c_int),
        "nebw_model_set_int8_operand": ([vp, C.c_char_p, vp, vp, vp, i64, i64], C.c_int),
        "nebw_model_set_datapath": ([vp, i32], C.c_int),
        "nebw_model_set_graphs": ([vp, i32], C.c_int),
        "nebw_rope_freqs": ([C.c_double, i32, C.POINTER(RopeScaling), C.POINTER(C.c_double),
                             C.POINTER(C.c_double)], C.c_int),
        "nebw_stage_rope": ([vp, C.POINTER(C.c_double), i32, i64, C.c_double,
                             C.POINTER(C.c_uint64)], C.c_int),
        "nebw_row_positions": ([vp, vp, vp, i32, i32, vp, vp], C.c_int),
        "nebw_packed_positions": ([vp, vp, vp, i32, i32, i64, vp, vp], C.c_int),
        "nebw_rope": ([vp, C.POINTER(Heads), C.POINTER(Heads), C.c_int, i64, vp, i32, C.c_uint64,
                       C.c_int, vp, vp], C.c_int),
        "nebw_qk_norm_rope": ([vp, C.POINTER(Heads), C.POINTER(Heads), C.c_int, i64, vp, i32,
                               C.c_int, C.c_float, C.c_uint64, C.c_int, vp, vp], C.c_int),
        "nebw_stage_experts": ([vp, vp, C.c_int, i32, i64, i64, C.c_int, vp,
                                C.POINTER(C.c_uint64)], C.c_int),
        "nebw_moe_route_workspace": ([i64, i32, i32], i64),
        "nebw_moe_route": ([vp, vp, C.c_int, i64, i64, vp, i32, i32, C.c_int, C.c_int, C.c_float,
                            vp, vp, vp, vp, vp, vp, i64, vp], C.c_int),
        "nebw_gemm_grouped": ([vp, C.c_uint64, vp, i64, vp, vp, i64, i64, i64, vp, C.c_int, vp,
                               C.c_int, vp], C.c_int),
        "nebw_moe_combine": ([vp, vp, C.c_int, i64, vp, vp, i64, vp, i32, i64, vp, vp, C.c_int,
                              vp], C.c_int),
        "nebw_pack_checkpoint": ([C.c_char_p, C.c_char_p, C.c_char_p, i32, i32,
                                  C.POINTER(C.c_uint64)], C.c_int),
        "nebw_comm_unique_id": ([vp], C.c_int),
        "nebw_comm_init_rank": ([vp, i32, i32, vp, C.c_double, C.POINTER(vp)], C.c_int),
        "nebw_comm_init_all": ([i32, C.POINTER(vp), C.c_double, C.POINTER(vp)], C.c_int),
        "nebw_comm_destroy": ([vp], C.c_int),
        "nebw_comm_size": ([vp, C.POINTER(i32), C.POINTER(i32)], C.c_int),
        "nebw_comm_sync": ([vp, vp], C.c_int),
        "nebw_shard_plan": ([vp, i32, i32, vp, vp], C.c_int),
        "nebw_shard_order": ([vp, i32, i32, vp], C.c_int),
        "nebw_gather_rows": ([vp, vp, vp, i32, vp, i32, vp], C.c_int),
        "nebw_encode_shard_gather": ([vp, vp, vp, vp, i32, i32, vp, vp, vp, vp], C.c_int),
        "nebw_encode_sharded": ([vp, vp, vp, vp, i32, i32, vp], C.c_int),
        "nebw_encode_multi": ([i32, C.POINTER(vp), C.POINTER(vp), vp, vp, i32, i32, vp], C.c_int),
    }
    for name, (args, res) in sig.items():
        f = getattr(L, name)
        f.argtypes = args
        f.restype = res
    _lib = L
    return L


def _check(rc: int):
    if rc != 0:
        raise NebwError(rc, lib().nebw_last_error().decode())


def _addr(x):
    """Device/host address of a torch tensor, numpy array, int or None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    try:
        return x.data_ptr()
    except AttributeError:
        pass
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    raise TypeError(f"cannot take the address of {type(x)}")


_INT32 = _FLOAT32 = _BFLOAT16 = None  # torch's dtypes, once it is in use


def _torch_dtypes():
    global _INT32, _FLOAT32, _BFLOAT16
    import torch
    _INT32, _FLOAT32, _BFLOAT16 = torch.int32, torch.float32, torch.bfloat16


def _dtype(t) -> int:
    """F32 or BF16 of a torch tensor."""
    if _BFLOAT16 is None:
        _torch_dtypes()
    if t.dtype is _BFLOAT16:
        return BF16
    if t.dtype is _FLOAT32:
        return F32
    raise TypeError(f"fp32 or bf16 is required, not {t.dtype}")


CUDA_STREAM_LEGACY = 1  # cudaStreamLegacy: the legacy default stream's handle


def _stream(s):
    """cudaStream_t for the C ABI.  None -> the library's own stream (NULL);
    a torch stream -> its handle, with torch's legacy default stream (handle
    0) passed as cudaStreamLegacy so that it is not read as NULL."""
    if s is None:
        return None
    h = s if isinstance(s, int) else s.cuda_stream
    return h if h != 0 else CUDA_STREAM_LEGACY


class Device:
    """One GPU (nebw_dev)."""

    def __init__(self, index: int = 0, torch_stream: bool = False):
        """torch_stream: op calls that name no stream run on torch's current
        stream (so they are ordered with the torch ops that made their
        buffers) instead of on the handle's own stream."""
        h = C.c_void_p()
        _check(lib().nebw_open(index, C.byref(h)))
        self.h = h
        self.index = index
        self.torch_stream = torch_stream
        self._experts = {}  # handle -> (experts, K, N, columns of the output)
        self._raw_stream = None
        if torch_stream:
            # the current stream's handle without a Stream object around it
            # (0.1 against 1.4 us of every call), where torch has the function
            import torch
            self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

    def _s(self, stream):
        if stream is not None:
            return _stream(stream)
        if self._raw_stream is not None:
            return self._raw_stream(self.index) or CUDA_STREAM_LEGACY
        if self.torch_stream:
            import torch
            return _stream(torch.cuda.current_stream(self.index))
        return None

    def _typed(self, x, name: str, n: int = 0, width: int = 0):
        """Device address of n contiguous values of a dtype: a torch tensor of
        another dtype, with gaps, in host memory, on another GPU or with fewer
        values is refused (its bytes would be read as other numbers, or what
        lies behind them), and so are more than n in rows of another width, if
        one is given (they would be read as rows of that width)."""
        if x is None or isinstance(x, int):
            return x
        import torch
        if (x.dtype is not getattr(torch, name) or x.get_device() != self.index
                or not x.is_contiguous()):
            raise TypeError(f"contiguous {name} values on the handle's GPU are required")
        have = x.numel()
        if have != n:
            if have < n:
                raise ValueError(f"{have} {name} values where {n} are read or written")
            if width:
                self._wide(x, width)
        return x.data_ptr()

    @staticmethod
    def _wide(x, width: int):
        if x.dim() > 1 and x.size(-1) != width:
            raise ValueError(f"rows of {x.size(-1)} values where they are of {width}")

    # The two below are _typed without its lookups (a short call has half a
    # dozen of them).
    def _i32(self, x, n: int = 0, width: int = 0):
        if x is None or x.__class__ is int:
            return x
        if x.dtype is _INT32 and x.get_device() == self.index and x.is_contiguous():
            have = x.numel()
            if have == n or (have > n and not width):
                return x.data_ptr()
        _torch_dtypes()
        return self._typed(x, "int32", n, width)

    def _f32(self, x, n: int = 0, width: int = 0):
        if x is None or x.__class__ is int:
            return x
        if x.dtype is _FLOAT32 and x.get_device() == self.index and x.is_contiguous():
            have = x.numel()
            if have == n or (have > n and not width):
                return x.data_ptr()
        _torch_dtypes()
        return self._typed(x, "float32", n, width)

    def close(self):
        if self.h:
            lib().nebw_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def sync(self):
        if self.torch_stream:
            import torch
            torch.cuda.current_stream().synchronize()
        _check(lib().nebw_sync(self.h))

    ATTN_MMA, ATTN_TCGEN05 = 0, 1

    def set_attention_kernel(self, kind: int):
        _check(lib().nebw_set_attention_kernel(self.h, kind))

    def check_bounded_wait(self, limit_ns: int) -> bool:
        """True if the probe's wait ran out (nebw_check_bounded_wait)."""
        e = C.c_int32()
        _check(lib().nebw_check_bounded_wait(self.h, limit_ns, C.byref(e)))
        return bool(e.value)

    def info(self):
        sm, ma, mi = C.c_int(), C.c_int(), C.c_int()
        _check(lib().nebw_device_info(self.h, C.byref(sm), C.byref(ma), C.byref(mi)))
        return {"sm_count": sm.value, "cc": (ma.value, mi.value)}

    # ---- weights and ops -------------------------------------------------
    def stage_weight(self, w_kn: np.ndarray) -> int:
        w = np.ascontiguousarray(w_kn)
        dt = F32 if w.dtype == np.float32 else BF16
        if w.dtype not in (np.float32, np.uint16):
            raise TypeError("weights are fp32, or bf16 bit patterns as uint16")
        K, N = w.shape
        hnd = C.c_uint64()
        _check(lib().nebw_stage_weight(self.h, w.ctypes.data, dt, K, N, C.byref(hnd)))
        return hnd.value

    def stage_weight_i8(self, w_kn: np.ndarray) -> int:
        """An int8 [K, N] GEMM operand (nebw_stage_weight_i8)."""
        w = np.ascontiguousarray(w_kn, np.int8)
        K, N = w.shape
        hnd = C.c_uint64()
        _check(lib().nebw_stage_weight_i8(self.h, w.ctypes.data, K, N, C.byref(hnd)))
        return hnd.value

    def gemm_i8(self, weight, A, sa, M, K, N, ws, C_out, bias=None, act=ACT_NONE, stream=None,
                c_dtype=F32):
        """C = dequant(A . W) (nebw_gemm_i8_ex): fp32 C, or bf16 RNE with c_dtype BF16."""
        _check(lib().nebw_gemm_i8_ex(self.h, weight, _addr(A), _addr(sa), M, K, N, _addr(ws),
                                     _addr(bias), act, _addr(C_out), c_dtype, self._s(stream)))

    def quantise_rows(self, x, rows, K, ias, q, scale, stream=None):
        """quantise_a_int8 per row; x fp32, or a torch bf16 tensor (widened exactly)."""
        fn = (lib().nebw_quantise_rows_bf16 if str(getattr(x, "dtype", "")) == "torch.bfloat16"
              else lib().nebw_quantise_rows)
        _check(fn(self.h, _addr(x), rows, K, _addr(ias), _addr(q), _addr(scale), self._s(stream)))

    def layernorm_quant(self, x, gamma, beta, rows, H, y=None, ias=None, q=None, scale=None,
                        eps=1e-12, stream=None):
        """add_norm_quant: x = LN(x + y) in place (y fp32 or None), then the rows
        quantised with ias into q / scale when q is given."""
        _check(lib().nebw_layernorm_quant(self.h, _addr(x), _addr(y), _addr(gamma), _addr(beta),
                                          eps, rows, H, _addr(ias), _addr(q), _addr(scale),
                                          self._s(stream)))

    def release_weight(self, handle: int):
        _check(lib().nebw_release_weight(self.h, handle))
        self._experts.pop(handle, None)

    def gemm(self, weight, A, M, K, N, C_out, bias=None, residual=None, act=ACT_NONE,
             c_dtype=BF16, stream=None):
        _check(lib().nebw_gemm(self.h, weight, _addr(A), M, K, N, _addr(bias), _addr(residual),
                               act, _addr(C_out), c_dtype, self._s(stream)))

    def layernorm(self, x, gamma, beta, rows, H, y=None, a_bf16=None, eps=1e-12, stream=None,
                  y_dtype=None):
        """x = LN(x + y) in place; y_dtype defaults to y's own (torch bf16 -> BF16, else F32)."""
        if y_dtype is None:
            y_dtype = BF16 if str(getattr(y, "dtype", "")) == "torch.bfloat16" else F32
        _check(lib().nebw_layernorm(self.h, _addr(x), _addr(y), y_dtype, _addr(gamma),
                                    _addr(beta), eps, rows, H, _addr(a_bf16), self._s(stream)))

    def attention(self, qkv, rows, seq_off, seq_len, B, max_len, heads, head_dim, ctx, stream=None):
        _check(lib().nebw_attention(self.h, _addr(qkv), rows, _addr(seq_off), _addr(seq_len), B,
                                    max_len, heads, head_dim, _addr(ctx), self._s(stream)))

    def pack_offsets(self, len_in, B, S, len_out, seq_off, stream=None):
        _check(lib().nebw_pack_offsets(self.h, _addr(len_in), B, S, _addr(len_out),
                                       _addr(seq_off), self._s(stream)))

    def embed_ln(self, ids, seq_off, seq_len, B, S, word, vocab, pos, typ, gamma, beta, H, x,
                 a_bf16=None, eps=1e-12, stream=None):
        _check(lib().nebw_embed_ln(self.h, _addr(ids), _addr(seq_off), _addr(seq_len), B, S,
                                   _addr(word), vocab, _addr(pos), _addr(typ), _addr(gamma),
                                   _addr(beta), eps, H, _addr(x), _addr(a_bf16), self._s(stream)))

    def pool_l2(self, h, seq_off, seq_len, B, H, pooling, out, l2=True, stream=None):
        _check(lib().nebw_pool_l2(self.h, _addr(h), _addr(seq_off), _addr(seq_len), B, H,
                                  pooling, int(l2), _addr(out), self._s(stream)))

    def narrow_bf16(self, x, n, y, stream=None):
        _check(lib().nebw_narrow_bf16(self.h, _addr(x), n, _addr(y), self._s(stream)))

    # ---- rotary positions, head norms --------------------------------------
    def stage_rope(self, inv_freq, max_pos: int, scale: float = 1.0) -> int:
        """The rotary table of positions [0, max_pos) (nebw_stage_rope)."""
        f = np.ascontiguousarray(inv_freq, np.float64)
        hnd = C.c_uint64()
        _check(lib().nebw_stage_rope(self.h, f.ctypes.data_as(C.POINTER(C.c_double)), f.size,
                                     max_pos, scale, C.byref(hnd)))
        return hnd.value

    def row_positions(self, seq_off, seq_len, B, max_len, pos, stream=None, rows=None):
        """The packed rows' positions in their sequences (nebw_packed_positions):
        pos has `rows` entries, all of a tensor's if not given (an address
        needs them)."""
        if rows is None:
            if pos is None or pos.__class__ is int:
                raise ValueError("positions at an address need their number")
            rows = pos.numel()
        _check(lib().nebw_packed_positions(self.h, self._i32(seq_off, B), self._i32(seq_len, B), B,
                                           max_len, rows, self._i32(pos, rows), self._s(stream)))

    def _heads_dtype(self, q, k, dtype, rows, head_dim):
        """The dtype of heads made by Heads.of, which must hold the rows and
        have head_dim elements each, or the one given."""
        for h in (q, k):
            d = getattr(h, "dtype", None)
            if d is not None:
                if dtype is not None and dtype != d:
                    raise TypeError("query and key heads of different dtypes")
                if h.gpu != self.index:
                    raise TypeError("heads on the handle's GPU are required")
                if rows > h.rows or head_dim != h.head_dim:
                    if rows > h.rows or head_dim > h.head_dim:
                        raise ValueError(f"{rows} rows of {h.heads} x {head_dim} in heads of "
                                         f"[{h.rows}, {h.heads} x {h.head_dim}]")
                    # (a norm's weights have their length too)
                    raise NebwError(1, f"heads of {h.head_dim} elements are more than head_dim "
                                       f"{head_dim}")
                dtype = d
        return BF16 if dtype is None else dtype

    def rope(self, q, k, rows, head_dim, rope, pos, layout=ROPE_HALF, dtype=None, rows_dev=None,
             stream=None):
        """Rotary positions on the heads q and k (Heads, either may be None) (nebw_rope)."""
        dtype = self._heads_dtype(q, k, dtype, rows, head_dim)
        _check(lib().nebw_rope(self.h, q, k, dtype, rows, self._i32(rows_dev, 1), head_dim, rope,
                               layout, self._i32(pos, rows), self._s(stream)))

    def qk_norm_rope(self, q, k, rows, head_dim, norm=HEADNORM_RMS, eps=1e-6, rope=0, pos=None,
                     layout=ROPE_HALF, dtype=None, rows_dev=None, stream=None):
        """A norm of every head, then the rotation (rope 0: none) (nebw_qk_norm_rope)."""
        dtype = self._heads_dtype(q, k, dtype, rows, head_dim)
        _check(lib().nebw_qk_norm_rope(self.h, q, k, dtype, rows, self._i32(rows_dev, 1), head_dim,
                                       norm, eps, rope, layout, self._i32(pos, rows),
                                       self._s(stream)))

    # ---- experts -----------------------------------------------------------
    def stage_experts(self, w_ekn, gated: bool = False, stream=None) -> int:
        """Expert weights [experts, K, N] (nebw_stage_experts): numpy fp32, or
        bf16 bits as uint16, or a contiguous fp32 / bf16 torch tensor."""
        if isinstance(w_ekn, np.ndarray):
            w = np.ascontiguousarray(w_ekn)
            if w.dtype not in (np.float32, np.uint16):
                raise TypeError("weights are fp32, or bf16 bit patterns as uint16")
            dt = F32 if w.dtype == np.float32 else BF16
        else:
            w, dt = w_ekn, _dtype(w_ekn)
            if not w.is_contiguous():  # a copy would be made on torch's stream, not on this one
                raise ValueError("contiguous expert weights are required")
        E, K, N = w.shape
        hnd = C.c_uint64()
        _check(lib().nebw_stage_experts(self.h, _addr(w), dt, E, K, N, int(gated),
                                        self._s(stream), C.byref(hnd)))
        self._experts[hnd.value] = (E, K, N, N // 2 if gated else N)
        return hnd.value

    def moe_route(self, logits, rows, experts, top_k, ids, weights, group_off, row_src, row_dst,
                  workspace, score=ROUTE_SOFTMAX, renorm=False, scale=1.0, rows_dev=None,
                  stream=None):
        """The top_k experts of each row of logits (a 2-D fp32 / bf16 torch
        tensor, its row stride kept) and the rows grouped by expert
        (nebw_moe_route).  workspace: a tensor of moe_route_workspace bytes,
        or None where that is 0."""
        shape = logits.shape
        if len(shape) != 2 or logits.stride(1) != 1 or shape[1] < experts:
            raise ValueError("logits are rows of at least `experts` adjacent values")
        if shape[0] < rows:
            raise ValueError("fewer logit rows than rows")
        ws, ws_bytes = None, 0
        if workspace is not None:
            ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if (logits.get_device() != self.index or ws_bytes
                and (workspace.get_device() != self.index or not workspace.is_contiguous())):
            raise TypeError("logits and a contiguous workspace on the handle's GPU are required")
        stride = logits.stride(0) if rows > 1 else experts  # one row: torch may give any
        n = rows * top_k
        wide = top_k if 0 < top_k <= experts and top_k <= MAX_TOP_K else 0  # or refused below
        _check(lib().nebw_moe_route(self.h, logits.data_ptr(), _dtype(logits), stride, rows,
                                    self._i32(rows_dev, 1), experts, top_k, score, int(renorm),
                                    scale, self._i32(ids, n, wide), self._f32(weights, n, wide),
                                    self._i32(group_off, experts + 1), self._i32(row_src, n),
                                    self._i32(row_dst, n, wide), ws, ws_bytes,
                                    self._s(stream)))

    def gemm_grouped(self, weight, A, a_rows, group_off, rows, K, N, C_out, row_src=None,
                     bias=None, act=ACT_NONE, c_dtype=BF16, stream=None):
        """One product per expert over its group of rows (nebw_gemm_grouped)."""
        # (a handle that is not there is refused below)
        e, k, n, width = self._experts.get(weight, (0, 0, 0, 0))
        try:
            out = self._typed(C_out, "bfloat16" if c_dtype == BF16 else "float32", rows * width,
                              width)
            A = self._typed(A, "bfloat16", a_rows * k, k)
            bias = self._f32(bias, e * n, n)
        except ValueError:
            # what the library refuses without the operands is said first
            _check(lib().nebw_gemm_grouped(self.h, weight, None, 0, None, None, 0, K, N, None, act,
                                           None, c_dtype, None))
            raise
        _check(lib().nebw_gemm_grouped(self.h, weight, A, a_rows, self._i32(row_src, rows),
                                       self._i32(group_off, e + 1), rows, K, N, bias, act, out,
                                       c_dtype, self._s(stream)))

    def moe_combine(self, y, row_dst, weights, rows, top_k, H, out, residual=None, rows_dev=None,
                    stream=None):
        """The experts' rows y (torch, [.., H]) weighted and summed per row
        (nebw_moe_combine)."""
        if (y.get_device() != self.index or out.get_device() != self.index
                or not (y.is_contiguous() and out.is_contiguous())):
            raise TypeError("contiguous expert rows and output on the handle's GPU are required")
        y_rows, n = y.shape[0], rows * top_k
        if H > 0:  # (other widths are refused below)
            if y.numel() != y_rows * H:  # not rows of H: of another width, or in more dimensions
                self._wide(y, H)
                y_rows = y.numel() // H
            have = out.numel()
            if have != rows * H:
                if have < rows * H:
                    raise ValueError(f"output {tuple(out.shape)} for {rows} rows of {H}")
                self._wide(out, H)
        wide = top_k if 0 < top_k <= MAX_TOP_K else 0
        _check(lib().nebw_moe_combine(self.h, y.data_ptr(), _dtype(y), y_rows,
                                      self._i32(row_dst, n, wide), self._f32(weights, n, wide),
                                      rows, self._i32(rows_dev, 1), top_k, H,
                                      self._f32(residual, rows * H, H), out.data_ptr(),
                                      _dtype(out), self._s(stream)))


ROPE_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}


def rope_freqs(theta: float, rot_dim: int, scaling: str = "none", factor: float = 1.0,
               orig_len: int = 0, fast: float = 0.0, slow: float = 0.0, attn_scale: float = 0.0):
    """(inv_freq [rot_dim / 2], scale) of rotary positions, scaled for
    positions past the trained length (nebw_rope_freqs)."""
    inv = np.empty(max(1, rot_dim // 2), np.float64)
    scale = C.c_double()
    s = RopeScaling(ROPE_SCALINGS[scaling], 0, orig_len, factor, fast, slow, attn_scale)
    _check(lib().nebw_rope_freqs(theta, rot_dim, C.byref(s),
                                 inv.ctypes.data_as(C.POINTER(C.c_double)), C.byref(scale)))
    return inv, scale.value


def moe_route_workspace(rows: int, experts: int, top_k: int) -> int:
    """Bytes of device workspace of Device.moe_route."""
    n = lib().nebw_moe_route_workspace(rows, experts, top_k)
    if n < 0:
        raise NebwError(1, lib().nebw_last_error().decode())
    return n


class Model:
    """A staged BERT encoder on one Device (nebw_model)."""

    def __init__(self, dev: Device, handle):
        self.dev = dev
        self.h = handle
        cfg = Config()
        _check(lib().nebw_model_get_config(self.h, C.byref(cfg)))
        self.cfg = cfg

    @classmethod
    def from_weights(cls, dev: Device, w, max_seq_len: int = 512, activation: int = ACT_GELU8):
        """Stage a nebw.synth.BertWeights (container layout) on `dev`."""
        gated = getattr(w, "gated", "")
        cfg = Config(num_layers=w.layers, hidden=w.hidden, num_heads=w.heads,
                     head_dim=w.head_dim, intermediate=w.ffn, vocab_size=w.vocab,
                     max_seq_len=max_seq_len, type_vocab_size=w.typ.shape[0],
                     pooling=POOL_CLS if w.cls_pool else POOL_MEAN, l2_normalize=1,
                     activation=ACT_GELU_ERF if getattr(w, "gelu_erf", False) else activation,
                     layer_norm_eps=1e-12, gated_ffn=int(bool(gated)),
                     gated_act=GATE_GELU_ERF if gated == "geglu" else GATE_SILU,
                     rope=int(getattr(w, "rope", False)),
                     rope_theta=float(getattr(w, "rope_theta", 0.0)))
        h = C.c_void_p()
        _check(lib().nebw_model_create(dev.h, C.byref(cfg), C.byref(h)))
        m = cls(dev, h)
        try:
            freq = getattr(w, "rope_inv_freq", ())
            if len(freq):  # held as float32, as the reference reads them
                f = np.ascontiguousarray(np.asarray(freq, np.float32).astype(np.float64))
                _check(lib().nebw_model_set_rope_freq(
                    m.h, f.ctypes.data_as(C.POINTER(C.c_double)), len(f)))
            for name, arr in w.tensors():
                a = np.ascontiguousarray(arr, np.float32)
                rows, cols = (a.shape[0], a.shape[1]) if a.ndim == 2 else (1, a.shape[0])
                if name == "embeddings.position":
                    a = np.ascontiguousarray(a[:max_seq_len])
                    rows = a.shape[0]
                _check(lib().nebw_model_set_tensor(m.h, name.encode(), a.ctypes.data, F32, rows,
                                                   cols))
        except Exception:
            m.close()
            raise
        return m

    @classmethod
    def from_npue(cls, dev: Device, path):
        h = C.c_void_p()
        _check(lib().nebw_model_load_npue(dev.h, str(path).encode(), C.byref(h)))
        return cls(dev, h)

    def set_tensor(self, name: str, arr):
        """(Re)stage one tensor by its container name, fp32 (nebw_model_set_tensor)."""
        a = np.ascontiguousarray(arr, np.float32)
        rows, cols = (a.shape[0], a.shape[1]) if a.ndim == 2 else (1, a.shape[0])
        _check(lib().nebw_model_set_tensor(self.h, name.encode(), a.ctypes.data, F32, rows, cols))

    DATAPATHS = {"bf16": 0, "i8": 1}

    def set_datapath(self, datapath: str):
        """"bf16" (default) or "i8": the int8 array path of an int8 container
        (nebw_model_set_datapath)."""
        _check(lib().nebw_model_set_datapath(self.h, self.DATAPATHS[datapath]))

    def set_graphs(self, on: bool = True):
        """encode() replays each (B, S) shape's pass as a CUDA graph (nebw_model_set_graphs)."""
        _check(lib().nebw_model_set_graphs(self.h, int(bool(on))))

    def set_int8_operand(self, name: str, kn, wscale, asmooth):
        """An int8 GEMM operand [K, N] with its .wscale [N] and .asmooth [K]."""
        q = np.ascontiguousarray(kn, np.int8)
        ws = np.ascontiguousarray(wscale, np.float32)
        asm = np.ascontiguousarray(asmooth, np.float32)
        K, N = q.shape
        _check(lib().nebw_model_set_int8_operand(self.h, name.encode(), q.ctypes.data,
                                                 ws.ctypes.data, asm.ctypes.data, K, N))

    def close(self):
        if self.h:
            lib().nebw_model_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def hidden(self) -> int:
        return self.cfg.hidden

    def launch_count(self, seq: int = 0) -> int:
        return lib().nebw_encode_launch_count(self.h, seq)

    KERNEL_KINDS = ("pack", "embed_ln", "gemm_qkv", "attention", "gemm_ao", "layernorm",
                    "gemm_up", "gemm_down", "pool")

    def profile(self, enable: bool = True):
        _check(lib().nebw_model_profile(self.h, int(enable)))

    def profile_collect(self) -> dict:
        """{kind: (launches, device ms)} since the last collect."""
        n = len(self.KERNEL_KINDS)
        launches = (C.c_int64 * n)()
        ms = (C.c_double * n)()
        _check(lib().nebw_model_profile_collect(self.h, launches, ms))
        return {k: (int(launches[i]), float(ms[i])) for i, k in enumerate(self.KERNEL_KINDS)}

    def encode(self, ids: np.ndarray, lens: np.ndarray) -> np.ndarray:
        """Host in, host out: ids [B, S] int32, lens [B] int32 -> [B, hidden]."""
        ids = np.ascontiguousarray(ids, np.int32)
        lens = np.ascontiguousarray(lens, np.int32)
        B, S = ids.shape
        out = np.empty((B, self.hidden), np.float32)
        _check(lib().nebw_encode(self.h, ids.ctypes.data, lens.ctypes.data, B, S, out.ctypes.data))
        return out

    def encode_into(self, ids, lens, out, B: int, S: int, host=False, stream=None):
        """Host or device buffers by address; the device form is asynchronous."""
        if host:
            _check(lib().nebw_encode(self.h, _addr(ids), _addr(lens), B, S, _addr(out)))
        else:
            _check(lib().nebw_encode_device(self.h, _addr(ids), _addr(lens), B, S, _addr(out),
                                            _stream(stream)))


class VitModel:
    """A staged ViT encoder (container arch vit_patch16_prenorm_gelu) on one
    device: images [n, C, S, S] fp32 -> the CLS row after the final
    LayerNorm, [n, hidden] fp32."""

    KERNEL_KINDS = Model.KERNEL_KINDS

    def __init__(self, dev: Device, handle):
        self.dev = dev
        self.h = handle
        cfg = VitConfig()
        _check(lib().nebw_vit_get_config(self.h, C.byref(cfg)))
        self.cfg = cfg

    @classmethod
    def from_weights(cls, dev: Device, w):
        """Stage a nebw.synth.VitWeights on `dev`."""
        a = w.arch
        cfg = VitConfig(num_layers=w.layers, hidden=a.hidden, num_heads=a.heads,
                        head_dim=a.head_dim, intermediate=a.ffn, image_size=a.image_size,
                        patch_size=a.patch_size, num_channels=a.channels,
                        layer_norm_eps=a.ln_eps)
        h = C.c_void_p()
        _check(lib().nebw_vit_create(dev.h, C.byref(cfg), C.byref(h)))
        m = cls(dev, h)
        try:
            for name, arr in w.tensors():
                x = np.ascontiguousarray(arr, np.float32)
                rows, cols = (x.shape[0], x.shape[1]) if x.ndim == 2 else (1, x.shape[0])
                _check(lib().nebw_vit_set_tensor(m.h, name.encode(), x.ctypes.data, F32, rows,
                                                 cols))
        except Exception:
            m.close()
            raise
        return m

    @classmethod
    def from_npue(cls, dev: Device, path):
        h = C.c_void_p()
        _check(lib().nebw_vit_load_npue(dev.h, str(path).encode(), C.byref(h)))
        return cls(dev, h)

    def close(self):
        if self.h:
            lib().nebw_vit_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def hidden(self) -> int:
        return self.cfg.hidden

    def launch_count(self) -> int:
        return lib().nebw_vit_launch_count(self.h)

    def profile(self, enable: bool = True):
        _check(lib().nebw_vit_profile(self.h, int(enable)))

    def profile_collect(self) -> dict:
        n = len(self.KERNEL_KINDS)
        launches = (C.c_int64 * n)()
        ms = (C.c_double * n)()
        _check(lib().nebw_vit_profile_collect(self.h, launches, ms))
        return {k: (int(launches[i]), float(ms[i])) for i, k in enumerate(self.KERNEL_KINDS)}

    def encode(self, images: np.ndarray) -> np.ndarray:
        """Host in, host out."""
        images = np.ascontiguousarray(images, np.float32)
        out = np.empty((images.shape[0], self.hidden), np.float32)
        _check(lib().nebw_vit_encode(self.h, images.ctypes.data, images.shape[0],
                                     out.ctypes.data))
        return out

    def encode_into(self, images, out, n: int, host=False, stream=None):
        """Host or device buffers by address; the device form is asynchronous."""
        if host:
            _check(lib().nebw_vit_encode(self.h, _addr(images), n, _addr(out)))
        else:
            _check(lib().nebw_vit_encode_device(self.h, _addr(images), n, _addr(out),
                                                _stream(stream)))


# ---------------------------------------------------------------------------
# several GPUs (nebw_comm): the batch sharded, the embeddings gathered
# ---------------------------------------------------------------------------

COMM_ID_BYTES = 128


def shard_plan(lens, nranks: int):
    """(owner [B], counts [nranks]) of the library's length-balanced plan."""
    lens = np.ascontiguousarray(lens, np.int32)
    owner = np.empty(len(lens), np.int32)
    counts = np.empty(nranks, np.int32)
    _check(lib().nebw_shard_plan(lens.ctypes.data, len(lens), nranks, owner.ctypes.data,
                                 counts.ctypes.data))
    return owner, counts


def shard_order(owner, nranks: int) -> np.ndarray:
    """order[k] = request index of row k of the rank-major gather."""
    owner = np.ascontiguousarray(owner, np.int32)
    order = np.empty(len(owner), np.int32)
    _check(lib().nebw_shard_order(owner.ctypes.data, len(owner), nranks, order.ctypes.data))
    return order


def comm_unique_id() -> bytes:
    buf = (C.c_uint8 * COMM_ID_BYTES)()
    _check(lib().nebw_comm_unique_id(buf))
    return bytes(buf)


class Comm:
    """A rank of an NCCL communicator on one Device (nebw_comm)."""

    def __init__(self, dev: Device, handle):
        self.dev = dev
        self.h = handle
        n, r = C.c_int32(), C.c_int32()
        _check(lib().nebw_comm_size(self.h, C.byref(n), C.byref(r)))
        self.nranks, self.rank = n.value, r.value

    @classmethod
    def init_rank(cls, dev: Device, nranks: int, rank: int, uid: bytes, timeout_s: float = 60.0):
        if len(uid) != COMM_ID_BYTES:
            raise ValueError("a communicator id is 128 bytes")
        buf = (C.c_uint8 * COMM_ID_BYTES).from_buffer_copy(uid)
        h = C.c_void_p()
        _check(lib().nebw_comm_init_rank(dev.h, nranks, rank, buf, timeout_s, C.byref(h)))
        return cls(dev, h)

    @classmethod
    def init_all(cls, devs, timeout_s: float = 60.0):
        n = len(devs)
        dh = (C.c_void_p * n)(*[d.h.value for d in devs])
        out = (C.c_void_p * n)()
        _check(lib().nebw_comm_init_all(n, dh, timeout_s, out))
        return [cls(d, C.c_void_p(out[i])) for i, d in enumerate(devs)]

    def close(self):
        if self.h:
            rc = lib().nebw_comm_destroy(self.h)
            self.h = None
            _check(rc)

    def __del__(self):
        try:
            if self.h:
                lib().nebw_comm_destroy(self.h)
                self.h = None
        except Exception:
            pass

    def sync(self, stream=None):
        _check(lib().nebw_comm_sync(self.h, _stream(stream)))

    def gather_rows(self, rows, counts, H: int, out=None, root: int = 0, stream=None):
        counts = np.ascontiguousarray(counts, np.int32)
        _check(lib().nebw_gather_rows(self.h, _addr(rows), counts.ctypes.data, H, _addr(out), root,
                                      _stream(stream)))

    def encode_shard_gather(self, model: Model, ids, lens, b_r: int, S: int, counts, order=None,
                            out=None, stream=None):
        """Device-resident sharded pass (asynchronous; sync() waits)."""
        counts = np.ascontiguousarray(counts, np.int32)
        _check(lib().nebw_encode_shard_gather(model.h, self.h, _addr(ids), _addr(lens), b_r, S,
                                              counts.ctypes.data, _addr(order), _addr(out),
                                              _stream(stream)))

    def encode_sharded(self, model: Model, ids: np.ndarray, lens: np.ndarray, out=None):
        """Host buffers, synchronous; rank 0 gets [B, hidden] in request
        order (returned), the other ranks None."""
        ids = np.ascontiguousarray(ids, np.int32)
        lens = np.ascontiguousarray(lens, np.int32)
        B, S = ids.shape
        if self.rank == 0 and out is None:
            out = np.empty((B, model.hidden), np.float32)
        _check(lib().nebw_encode_sharded(model.h, self.h, ids.ctypes.data, lens.ctypes.data, B, S,
                                         _addr(out) if self.rank == 0 else None))
        return out if self.rank == 0 else None


def encode_multi(models, comms, ids: np.ndarray, lens: np.ndarray) -> np.ndarray:
    """One process, n GPUs (Comm.init_all): [B, hidden] in request order."""
    ids = np.ascontiguousarray(ids, np.int32)
    lens = np.ascontiguousarray(lens, np.int32)
    B, S = ids.shape
    n = len(models)
    out = np.empty((B, models[0].hidden), np.float32)
    mh = (C.c_void_p * n)(*[m.h.value for m in models])
    ch = (C.c_void_p * n)(*[c.h.value for c in comms])
    _check(lib().nebw_encode_multi(n, mh, ch, ids.ctypes.data, lens.ctypes.data, B, S,
                                   out.ctypes.data))
    return out


def pack_checkpoint(model_dir, out, layout: str = "tma_bf16", max_seq: int = 0,
                    fold_scale: bool = True) -> int:
    """The library's C++ packer (nebw_pack_checkpoint); returns the bytes written."""
    n = C.c_uint64()
    _check(lib().nebw_pack_checkpoint(str(model_dir).encode(), str(out).encode(),
                                      layout.encode(), int(max_seq), int(fold_scale),
                                      C.byref(n)))
    return n.value
