"""Python binding of the MI355X codec library (libboa_hip.so, C ABI in
include/boa_hip.h).

This is plumbing for tests, the benchmark and smoke(): the product is the C
ABI and the `boa` CLI.  Device buffers are passed as raw pointers (torch
tensors' data_ptr() or hipMalloc'd memory).  Importing the module never
falls back to anything: if the library is missing or fails to load, every
entry point raises.
"""
from __future__ import annotations

import ctypes as C
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libboa_hip.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "boa_hip.h")

BOA_OK = 0
(K_GEMM, K_SCAN, K_CONV, K_LN, K_CDF, K_CODER, K_DECODE, K_GEMM_SMALL, K_DEC_GEMM,
 K_DEC_SCAN, K_HEAD_CDF, K_DEC_LNGEMM) = range(12)
K_NAMES = ["gemm", "scan", "conv", "ln", "cdf", "coder", "decode", "gemm_small", "dec_gemm",
           "dec_scan", "head_cdf", "dec_lngemm"]
BOA_E_ARG, BOA_E_HIP, BOA_E_IO, BOA_E_FORMAT, BOA_E_STATE, BOA_E_NOMEM = -1, -2, -3, -4, -5, -6

# void (*)(void* user, int32_t phase, int64_t done_bytes, int64_t total_bytes)
PROGRESS_FN = C.CFUNCTYPE(None, C.c_void_p, C.c_int32, C.c_int64, C.c_int64)


class BoaError(RuntimeError):
    def __init__(self, msg, rc=None):
        super().__init__(msg)
        self.rc = rc


class Config(C.Structure):
    _fields_ = [("d_model", C.c_int32), ("n_layers", C.c_int32), ("d_state", C.c_int32),
                ("max_lanes", C.c_int32), ("tile", C.c_int32), ("precision", C.c_int32),
                ("temperature", C.c_float)]


class Rows(C.Structure):
    """boa_rows: a row tensor's first element and strides in elements."""
    _fields_ = [("d", C.c_void_p), ("lane_stride", C.c_int64), ("row_stride", C.c_int64)]


class Scan(C.Structure):
    """boa_scan: the inputs of the selective scan."""
    _fields_ = [("lanes", C.c_int32), ("T", C.c_int32), ("channels", C.c_int32),
                ("d_state", C.c_int32), ("precision", C.c_int32), ("d_lens", C.c_void_p),
                ("u", Rows), ("delta", Rows), ("z", Rows), ("b", Rows), ("c", Rows),
                ("d_A", C.c_void_p), ("d_D", C.c_void_p), ("d_delta_bias", C.c_void_p),
                ("d_state_in", C.c_void_p)]


class ScanGrads(C.Structure):
    """boa_scan_grads: the outputs of the scan's gradient."""
    _fields_ = [("du", Rows), ("ddelta", Rows), ("dz", Rows), ("db", Rows), ("dc", Rows),
                ("d_dA", C.c_void_p), ("d_dD", C.c_void_p), ("d_ddelta_bias", C.c_void_p),
                ("d_dstate_in", C.c_void_p)]


def build(clean: bool = False) -> str:
    """Compile libboa_hip.so and the boa CLI for gfx950 (hipcc)."""
    if clean:
        subprocess.run(["make", "-s", "-C", HERE, "clean"], check=True)
    subprocess.run(["make", "-s", "-C", HERE, "-j4"], check=True)
    return LIB_PATH


def declared_symbols() -> list[str]:
    """Function names declared in include/boa_hip.h."""
    txt = open(HEADER).read()
    txt = re.sub(r"/\*.*?\*/", "", txt, flags=re.S)
    return sorted(set(re.findall(r"\b(boa_[a-z0-9_]+)\s*\(", txt)))


_lib = None


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise BoaError(f"{LIB_PATH} is not built (run __graft_entry__.build())")
        L = C.CDLL(LIB_PATH)
        P, i32, i64, f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float
        sig = {
            "boa_create": (C.c_int, [C.POINTER(Config), C.POINTER(P)]),
            "boa_destroy": (None, [P]),
            "boa_last_error": (C.c_char_p, [P]),
            "boa_set_stream": (C.c_int, [P, P]),
            "boa_use_own_stream": (C.c_int, [P]),
            "boa_set_temperature": (C.c_int, [P, f32]),
            "boa_set_warm_start": (C.c_int, [P, i32]),
            "boa_set_progress": (C.c_int, [P, PROGRESS_FN, P]),
            "boa_decode_plan": (C.c_int, [P, i32, C.POINTER(i32), C.POINTER(i32)]),
            "boa_set_state_cache_budget": (C.c_int, [P, i64]),
            "boa_last_timings": (C.c_int, [P, C.POINTER(C.c_double), C.POINTER(C.c_double),
                                           C.POINTER(C.c_double)]),
            "boa_load_weights": (C.c_int, [P, C.c_char_p]),
            "boa_load_weights_mem": (C.c_int, [P, P, C.c_size_t]),
            "boa_weight_file_bytes": (i64, [i32, i32, i32, i32]),
            "boa_estimate_memory": (i64, [C.POINTER(Config), i64, i32]),
            "boa_reset_state": (C.c_int, [P, i32]),
            "boa_forward_chunk": (C.c_int, [P, P, i32, i32, P]),
            "boa_step_batch": (C.c_int, [P, P, i32, P, i32]),
            "boa_forward_chunk_noalloc": (C.c_int, [P, P, i32, i32, P]),
            "boa_device": (C.c_int, [P]),
            "boa_embed": (C.c_int, [P, P, i64, P, i32, i32, P, i32, i32, f32, C.POINTER(Rows)]),
            "boa_embed_grad": (C.c_int, [P, P, i64, P, i32, i32, C.POINTER(Rows), i32, i32, f32,
                                         P, P, i64]),
            "boa_embed_grad_work_bytes": (i64, [i32, i32, i32]),
            "boa_selective_scan": (C.c_int, [P, C.POINTER(Scan), C.POINTER(Rows), P, P, P, i64]),
            "boa_selective_scan_grad": (C.c_int, [P, C.POINTER(Scan), P, C.POINTER(Rows), P,
                                                  C.POINTER(ScanGrads), P, i64]),
            "boa_selective_scan_saved_floats": (i64, [i32, i32, i32, i32]),
            "boa_selective_scan_work_bytes": (i64, [i32, i32, i32, i32, i32]),
            "boa_next_byte_loss": (C.c_int, [P, C.POINTER(Rows), P, P, i64, P, i32, i32, i32, f32,
                                             P, P, C.POINTER(Rows), P, P, i64]),
            "boa_next_byte_loss_work_bytes": (i64, [i32, i32]),
            "boa_cdf_from_logits": (C.c_int, [P, P, P, i32, P]),
            "boa_cdf_from_probs": (C.c_int, [P, P, i32, i32, P]),
            "boa_rc_encode_cdf": (C.c_int, [P, P, P, i32, i32, P, i64, P]),
            "boa_rc_decode_cdf": (C.c_int, [P, P, i32, i32, P, i64, P, P]),
            "boa_compress_device": (C.c_int, [P, P, i64, i64, i32, P, i64, P, P, P]),
            "boa_num_chunks": (i64, [i64, i64, i32]),
            "boa_payload_bound_words": (i64, [i64, i64, i32]),
            "boa_decompress_device": (C.c_int, [P, P, P, P, P, i32, i64, i64, P]),
            "boa_compress_buffer": (C.c_int, [P, P, i64, i64, i32, C.POINTER(P), C.POINTER(i64)]),
            "boa_decompress_buffer": (C.c_int, [P, P, i64, C.POINTER(P), C.POINTER(i64)]),
            "boa_compress_file": (C.c_int, [P, C.c_char_p, C.c_char_p, i64, i32]),
            "boa_decompress_file": (C.c_int, [P, C.c_char_p, C.c_char_p]),
            "boa_free": (None, [P]),
            "boa_crc32": (C.c_uint32, [P, i64]),
            "boa_profile_enable": (C.c_int, [P, i32]),
            "boa_profile_reset": (C.c_int, [P]),
            "boa_profile_read": (C.c_int, [P, i32, C.POINTER(C.c_double), C.POINTER(i64),
                                           C.POINTER(C.c_double)]),
        }
        for name, (res, args) in sig.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _ptr(x):
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


# ---- training operators: tensors to C arguments
# (what the C entry points cannot see -- types, shapes, devices -- is checked
# here; sizes, strides, alignment and workspaces are checked there)
def _int32(*n):
    """Sizes that ctypes can pass as int32 (it would cut larger ones off)."""
    if max(n) >> 31 or min(n) < 0:
        raise ValueError(f"sizes out of range: {n}")
    return n


def _tensor(t, name, shape, dtype, device):
    """A dense tensor's pointer (None for None), of this shape and type on this device."""
    if t is None:
        return None
    if t.shape != shape or t.dtype != dtype:
        raise ValueError(f"{name}: want {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device:  # -1 on the CPU
        raise ValueError(f"{name} is on {t.device}, the context on cuda:{device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} has to be contiguous")
    return t.data_ptr()


def _rows(t, name, lanes, T, width, dtype, device):
    """A [lanes, T, width] tensor, dense in its last dimension, as a Rows."""
    if t.shape != (lanes, T, width) or t.dtype != dtype:
        raise ValueError(f"{name}: want {dtype} {(lanes, T, width)}, got {t.dtype} "
                         f"{tuple(t.shape)}")
    if t.get_device() != device:  # -1 on the CPU
        raise ValueError(f"{name} is on {t.device}, the context on cuda:{device}")
    ls, rs, one = t.stride()
    if one != 1 and width > 1:
        raise ValueError(f"{name} has to be dense in its last dimension")
    return Rows(t.data_ptr(), ls, rs)


def _bytes(t, name, device):
    """A uint8 [lanes, T] tensor, dense along T: (pointer, stride of a lane, lanes, T)."""
    torch = sys.modules["torch"]  # there is a tensor, so it is loaded
    if t.dim() != 2 or t.dtype != torch.uint8:
        raise ValueError(f"{name}: want uint8 [lanes, T], got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device:  # -1 on the CPU
        raise ValueError(f"{name} is on {t.device}, the context on cuda:{device}")
    (ls, one), (lanes, T) = t.stride(), t.shape
    if one != 1 and T > 1:
        raise ValueError(f"{name} has to be dense along T")
    if (lanes | T) >> 31:
        _int32(lanes, T)
    return t.data_ptr(), ls, lanes, T


def _precision(t, name):
    torch = sys.modules["torch"]  # there is a tensor, so it is loaded
    if t.dim() == 3:
        if t.dtype == torch.float32:
            return 0
        if t.dtype == torch.bfloat16:
            return 1
    raise ValueError(f"{name}: want float32 or bfloat16 [lanes, T, width], got {t.dtype} "
                     f"{tuple(t.shape)}")


def _work(t, device):
    """A workspace tensor of any type: (pointer, bytes)."""
    if t is None:
        return None, 0
    n = t.nbytes
    if n and (t.get_device() != device or not t.is_contiguous()):
        raise ValueError(f"the workspace has to be contiguous, on cuda:{device}")
    return (t.data_ptr() if n else None), n


def _size(n, what):
    if n < 0:
        raise ValueError(f"{what}: sizes out of range")
    return n


def embed_grad_work_bytes(lanes, T, width):
    return _size(lib().boa_embed_grad_work_bytes(*_int32(lanes, T, width)), "embed_grad")


def selective_scan_saved_floats(lanes, T, channels, d_state):
    return _size(lib().boa_selective_scan_saved_floats(*_int32(lanes, T, channels, d_state)),
                 "selective_scan")


def selective_scan_work_bytes(lanes, T, channels, d_state, grad=False):
    return _size(lib().boa_selective_scan_work_bytes(*_int32(lanes, T, channels, d_state),
                                                     int(grad)), "selective_scan")


def next_byte_loss_work_bytes(lanes, T):
    return _size(lib().boa_next_byte_loss_work_bytes(*_int32(lanes, T)), "next_byte_loss")


class Codec:
    """One context: weights, recurrent state and work buffers on one GPU."""

    def __init__(self, d_model, n_layers, d_state=16, max_lanes=64, tile=0, temperature=1.0,
                 precision="fp32"):
        prec = {"fp32": 0, "bf16": 1}[precision]
        self.cfg = Config(d_model, n_layers, d_state, max_lanes, tile, prec, temperature)
        h = C.c_void_p()
        rc = lib().boa_create(C.byref(self.cfg), C.byref(h))
        if rc != BOA_OK:
            raise BoaError(f"boa_create failed ({rc})")
        self.h = h
        self.device = lib().boa_device(h)

    def _check(self, rc, what):
        if rc != BOA_OK:
            raise BoaError(f"{what} failed ({rc}): {lib().boa_last_error(self.h).decode()}", rc)

    def close(self):
        if getattr(self, "h", None):
            lib().boa_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def load_weights(self, path):
        self._check(lib().boa_load_weights(self.h, str(path).encode()), "load_weights")

    def set_stream(self, stream_ptr):
        self._check(lib().boa_set_stream(self.h, stream_ptr), "set_stream")

    def reset_state(self, lanes):
        self._check(lib().boa_reset_state(self.h, lanes), "reset_state")

    def forward_chunk(self, d_tokens, lanes, T, d_logits):
        self._check(lib().boa_forward_chunk(self.h, _ptr(d_tokens), lanes, T, _ptr(d_logits)),
                    "forward_chunk")

    def forward_chunk_noalloc(self, d_tokens, lanes, T, d_logits):
        """boa_forward_chunk with its activations in the library's fixed
        per-GPU scratch array (no device allocation during the call)."""
        self._check(lib().boa_forward_chunk_noalloc(self.h, _ptr(d_tokens), lanes, T,
                                                    _ptr(d_logits)), "forward_chunk_noalloc")

    def step_batch(self, d_tokens, lanes, d_logits, add_bias=True):
        self._check(lib().boa_step_batch(self.h, _ptr(d_tokens), lanes, _ptr(d_logits),
                                         1 if add_bias else 0), "step_batch")

    def cdf_from_logits(self, d_logits, d_bias, rows, d_qcdf):
        self._check(lib().boa_cdf_from_logits(self.h, _ptr(d_logits), _ptr(d_bias), rows,
                                              _ptr(d_qcdf)), "cdf_from_logits")

    def cdf_from_probs(self, d_probs, rows, K, d_qcdf):
        self._check(lib().boa_cdf_from_probs(self.h, _ptr(d_probs), rows, K, _ptr(d_qcdf)),
                    "cdf_from_probs")

    def rc_encode_cdf(self, d_cdf, d_syms, n_sym, lanes, d_words, pitch_words, d_sizes):
        self._check(lib().boa_rc_encode_cdf(self.h, _ptr(d_cdf), _ptr(d_syms), n_sym, lanes,
                                            _ptr(d_words), pitch_words, _ptr(d_sizes)),
                    "rc_encode_cdf")

    def rc_decode_cdf(self, d_cdf, n_sym, lanes, d_words, pitch_words, d_sizes, d_syms):
        self._check(lib().boa_rc_decode_cdf(self.h, _ptr(d_cdf), n_sym, lanes, _ptr(d_words),
                                            pitch_words, _ptr(d_sizes), _ptr(d_syms)),
                    "rc_decode_cdf")

    # ---- training operators (boa_embed and the calls after it in boa_hip.h):
    # tensors on the context's device; row tensors [lanes, T, width], float32
    # or bfloat16, dense in their last dimension; d_lens int32 [lanes] or None
    def embed(self, d_tokens, d_table, d_out, scale=1.0, d_lens=None):
        """out = scale * table[tokens]; table [256, width] of out's type."""
        torch = sys.modules["torch"]
        dev = self.device
        tok, stride, lanes, T = _bytes(d_tokens, "tokens", dev)
        prec, dt, width = _precision(d_out, "out"), d_out.dtype, d_out.shape[2]
        self._check(lib().boa_embed(
            self.h, tok, stride, _tensor(d_lens, "lens", (lanes,), torch.int32, dev), lanes, T,
            _tensor(d_table, "table", (256, width), dt, dev), width, prec, scale,
            C.byref(_rows(d_out, "out", lanes, T, width, dt, dev))), "embed")

    def embed_grad(self, d_tokens, d_dout, d_dtable, d_work=None, scale=1.0, d_lens=None):
        """dtable (float32 [256, width]) = scale * sums of dout's rows by token."""
        torch = sys.modules["torch"]
        dev = self.device
        tok, stride, lanes, T = _bytes(d_tokens, "tokens", dev)
        prec, width = _precision(d_dout, "dout"), d_dout.shape[2]
        self._check(lib().boa_embed_grad(
            self.h, tok, stride, _tensor(d_lens, "lens", (lanes,), torch.int32, dev), lanes, T,
            C.byref(_rows(d_dout, "dout", lanes, T, width, d_dout.dtype, dev)), width, prec, scale,
            _tensor(d_dtable, "dtable", (256, width), torch.float32, dev),
            *_work(d_work, dev)), "embed_grad")

    def _scan_args(self, u, delta, z, b, c, A, D, delta_bias, state_in, lens):
        torch = sys.modules["torch"]
        dev, f32, prec = self.device, torch.float32, _precision(u, "u")
        (lanes, T, ch), dt = u.shape, u.dtype
        if A.dim() != 2:
            raise ValueError(f"A: want [channels, d_state], got {tuple(A.shape)}")
        n = A.shape[1]
        if (lanes | T | ch | n) >> 31:
            _int32(lanes, T, ch, n)
        return Scan(lanes, T, ch, n, prec, _tensor(lens, "lens", (lanes,), torch.int32, dev),
                    _rows(u, "u", lanes, T, ch, dt, dev),
                    _rows(delta, "delta", lanes, T, ch, dt, dev),
                    _rows(z, "z", lanes, T, ch, dt, dev),
                    _rows(b, "B", lanes, T, n, dt, dev), _rows(c, "C", lanes, T, n, dt, dev),
                    _tensor(A, "A", (ch, n), f32, dev), _tensor(D, "D", (ch,), f32, dev),
                    _tensor(delta_bias, "delta_bias", (ch,), f32, dev),
                    _tensor(state_in, "state_in", (lanes, ch, n), f32, dev))

    def selective_scan(self, d_u, d_delta, d_z, d_b, d_c, d_A, d_D, d_delta_bias, d_out,
                       d_work=None, d_state_in=None, d_state_out=None, d_lens=None, d_saved=None):
        """The gated recurrence; d_saved (selective_scan_saved_floats floats)
        keeps what its gradient starts from."""
        s, dev = self._scan_args(d_u, d_delta, d_z, d_b, d_c, d_A, d_D, d_delta_bias, d_state_in,
                                 d_lens), self.device
        out = _rows(d_out, "out", s.lanes, s.T, s.channels, d_u.dtype, dev)
        self._check(lib().boa_selective_scan(
            self.h, C.byref(s), C.byref(out),
            _tensor(d_state_out, "state_out", (s.lanes, s.channels, s.d_state), d_A.dtype, dev),
            self._saved(d_saved, s, dev), *_work(d_work, dev)), "selective_scan")

    def _saved(self, t, s, dev):
        if t is None:
            return None
        torch = sys.modules["torch"]
        n = lib().boa_selective_scan_saved_floats(s.lanes, s.T, s.channels, s.d_state)
        if t.numel() < n:
            raise ValueError(f"saved: want {n} floats, got {t.numel()}")
        return _tensor(t, "saved", t.shape, torch.float32, dev)

    def selective_scan_grad(self, d_u, d_delta, d_z, d_b, d_c, d_A, d_D, d_delta_bias, d_saved,
                            d_dout, d_du, d_ddelta, d_dz, d_db, d_dc, d_dA, d_dD, d_ddelta_bias,
                            d_work=None, d_state_in=None, d_dstate_out=None, d_dstate_in=None,
                            d_lens=None):
        """Gradients of selective_scan, from its inputs, its d_saved and the
        gradients of its outputs (d_dstate_out None: zero)."""
        s, dev = self._scan_args(d_u, d_delta, d_z, d_b, d_c, d_A, d_D, d_delta_bias, d_state_in,
                                 d_lens), self.device
        f32, dt, lanes, T, ch, n = d_A.dtype, d_u.dtype, s.lanes, s.T, s.channels, s.d_state
        dout = _rows(d_dout, "dout", lanes, T, ch, dt, dev)
        g = ScanGrads(_rows(d_du, "du", lanes, T, ch, dt, dev),
                      _rows(d_ddelta, "ddelta", lanes, T, ch, dt, dev),
                      _rows(d_dz, "dz", lanes, T, ch, dt, dev),
                      _rows(d_db, "dB", lanes, T, n, dt, dev),
                      _rows(d_dc, "dC", lanes, T, n, dt, dev),
                      _tensor(d_dA, "dA", (ch, n), f32, dev), _tensor(d_dD, "dD", (ch,), f32, dev),
                      _tensor(d_ddelta_bias, "ddelta_bias", (ch,), f32, dev),
                      _tensor(d_dstate_in, "dstate_in", (lanes, ch, n), f32, dev))
        self._check(lib().boa_selective_scan_grad(
            self.h, C.byref(s), self._saved(d_saved, s, dev), C.byref(dout),
            _tensor(d_dstate_out, "dstate_out", (lanes, ch, n), f32, dev), C.byref(g),
            *_work(d_work, dev)), "selective_scan_grad")

    def next_byte_loss(self, d_logits, d_targets, d_loss, d_work=None, d_bias=None, d_total=None,
                       d_dlogits=None, d_dbias=None, scale=1.0, d_lens=None):
        """loss [lanes, T] in nats, its sum, and scale times the gradients of
        the sum; dlogits may be logits."""
        torch = sys.modules["torch"]
        dev, f32 = self.device, torch.float32
        prec, dt = _precision(d_logits, "logits"), d_logits.dtype
        tgt, stride, lanes, T = _bytes(d_targets, "targets", dev)
        dx = None
        if d_dlogits is not None:
            dx = C.byref(_rows(d_dlogits, "dlogits", lanes, T, 256, dt, dev))
        self._check(lib().boa_next_byte_loss(
            self.h, C.byref(_rows(d_logits, "logits", lanes, T, 256, dt, dev)),
            _tensor(d_bias, "bias", (256,), f32, dev), tgt, stride,
            _tensor(d_lens, "lens", (lanes,), torch.int32, dev), lanes, T, prec, scale,
            _tensor(d_loss, "loss", (lanes, T), f32, dev), _tensor(d_total, "total", (1,), f32, dev),
            dx, _tensor(d_dbias, "dbias", (256,), f32, dev), *_work(d_work, dev)),
            "next_byte_loss")

    def compress_device(self, d_data, n, chunk_size, d_payload, cap_words, max_chunks=0):
        import numpy as np
        nc = lib().boa_num_chunks(n, chunk_size, max_chunks)
        lens = np.zeros(max(nc, 1), np.uint64)
        first = np.zeros(max(nc, 1), np.uint8)
        words = C.c_int64()
        self._check(lib().boa_compress_device(self.h, _ptr(d_data), n, chunk_size, max_chunks,
                                              _ptr(d_payload), cap_words, lens.ctypes.data,
                                              first.ctypes.data, C.byref(words)),
                    "compress_device")
        return lens[:nc], first[:nc], words.value

    def decompress_device(self, d_payload, offsets_words, stream_bytes, first, chunk_len,
                          last_len, d_out):
        import numpy as np
        offs = np.ascontiguousarray(offsets_words, np.uint64)
        lens = np.ascontiguousarray(stream_bytes, np.uint64)
        fb = np.ascontiguousarray(first, np.uint8)
        self._check(lib().boa_decompress_device(self.h, _ptr(d_payload), offs.ctypes.data,
                                                lens.ctypes.data, fb.ctypes.data, len(fb),
                                                chunk_len, last_len, _ptr(d_out)),
                    "decompress_device")

    def set_progress(self, fn):
        """fn(phase, done_bytes, total_bytes) during compress (phase 0) and
        decompress (phase 1); None turns the reports off."""
        if fn is None:
            self._progress = None
            self._check(lib().boa_set_progress(self.h, PROGRESS_FN(), None), "set_progress")
            return
        self._progress = PROGRESS_FN(lambda _u, ph, done, total: fn(ph, done, total))
        self._check(lib().boa_set_progress(self.h, self._progress, None), "set_progress")

    def decode_plan(self, lanes):
        """The decode step's schedule at `lanes` lanes: dict(cached_layers,
        fused_ln, persistent, fused_xproj, fused_head)."""
        a, f = C.c_int32(), C.c_int32()
        self._check(lib().boa_decode_plan(self.h, lanes, C.byref(a), C.byref(f)), "decode_plan")
        return dict(cached_layers=a.value, fused_ln=bool(f.value & 1),
                    persistent=bool(f.value & 2), fused_xproj=bool(f.value & 4),
                    fused_head=bool(f.value & 8))

    def last_timings(self):
        """(h2d_s, compute_s, d2h_s) of the last compress()/decompress() call."""
        a, b, c = C.c_double(), C.c_double(), C.c_double()
        self._check(lib().boa_last_timings(self.h, C.byref(a), C.byref(b), C.byref(c)),
                    "last_timings")
        return a.value, b.value, c.value

    def set_state_cache_budget(self, nbytes):
        self._check(lib().boa_set_state_cache_budget(self.h, int(nbytes)), "set_state_cache_budget")

    def set_warm_start(self, interleave_batch):
        """--warm-start (boa.cpp:310-319): 0 turns it off."""
        self._check(lib().boa_set_warm_start(self.h, int(interleave_batch)), "set_warm_start")

    def compress(self, data: bytes, chunk_size=4096, max_chunks=0) -> bytes:
        import numpy as np
        buf = np.frombuffer(data, np.uint8)
        out = C.c_void_p()
        n = C.c_int64()
        self._check(lib().boa_compress_buffer(self.h, buf.ctypes.data if len(data) else None,
                                              len(data), chunk_size, max_chunks, C.byref(out),
                                              C.byref(n)), "compress_buffer")
        res = C.string_at(out, n.value)
        lib().boa_free(out)
        return res

    def decompress(self, blob: bytes) -> bytes:
        import numpy as np
        buf = np.frombuffer(blob, np.uint8)
        out = C.c_void_p()
        n = C.c_int64()
        self._check(lib().boa_decompress_buffer(self.h, buf.ctypes.data, len(blob), C.byref(out),
                                                C.byref(n)), "decompress_buffer")
        res = C.string_at(out, n.value)
        lib().boa_free(out)
        return res

    def profile(self, on=True):
        self._check(lib().boa_profile_enable(self.h, 1 if on else 0), "profile_enable")

    def profile_reset(self):
        self._check(lib().boa_profile_reset(self.h), "profile_reset")

    def profile_read(self):
        out = {}
        for k, name in enumerate(K_NAMES):
            ms = C.c_double()
            n = C.c_int64()
            w = C.c_double()
            self._check(lib().boa_profile_read(self.h, k, C.byref(ms), C.byref(n), C.byref(w)),
                        "profile_read")
            out[name] = dict(ms=ms.value, launches=n.value, work=w.value)
        return out


def payload_bound_words(n, chunk_size, max_chunks=0):
    return lib().boa_payload_bound_words(n, chunk_size, max_chunks)
