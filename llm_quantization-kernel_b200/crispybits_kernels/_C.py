"""`crispybits_kernels._C` for B200: a ctypes shim over libcrispybits_b200.so.

The reference builds a pybind11/libtorch module of this name from
Crispybits/Kernel/csrc/bindings.cpp:32-40.  This module exposes the same seven functions with the
same positional signatures, so `ops.py` calls it unchanged, but the native side is a plain C ABI
(include/crispybits_b200.h): this file checks the tensors the way
Crispybits/Kernel/csrc/host_utils.h:49-87 does (failures raise RuntimeError, as TORCH_CHECK does),
allocates outputs and Split-K scratch with torch, and passes raw device pointers plus the current
CUDA stream across the boundary.

There is no CPU path here: importing this module without the built library raises ImportError, and
calling it with CPU tensors raises RuntimeError.
"""
from __future__ import annotations

import ctypes
import os
import threading
import weakref
from typing import Dict, List, Tuple

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(os.path.dirname(_HERE), "lib", "libcrispybits_b200.so")

if not os.path.exists(LIB_PATH):
    raise ImportError(f"{LIB_PATH} is not built; run `python llm_quantization-kernel_b200/build.py`")
_lib = ctypes.CDLL(LIB_PATH)

IS_EMULATOR = False
_vp, _i64, _int, _sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t


class _Weight(ctypes.Structure):
    """struct cb_weight of include/crispybits_b200.h"""
    _fields_ = [("packed", _vp), ("scales", _vp), ("zeros", _vp), ("bias", _vp), ("n", _i64)]


_WP = ctypes.POINTER(_Weight)
_lib.cb_last_error.restype = ctypes.c_char_p
_lib.cb_version.restype = ctypes.c_char_p
_lib.cb_gemv_scratch_bytes.restype = _sz
_lib.cb_gemv_scratch_bytes.argtypes = [_i64, _i64, _i64]
_lib.cb_packed_gemv.argtypes = [_vp, _i64, _WP, _vp, _i64, _int, _i64, _int, _i64, _i64, _int, _vp, _sz, _vp]
_lib.cb_fused_gate_up.argtypes = [_vp, _i64, _WP, _WP, _vp, _i64, _int, _i64, _int, _i64, _i64, _vp, _sz, _vp]
_lib.cb_fused_qkv.argtypes = [_vp, _i64, _WP, _WP, _WP, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _int, _i64,
                              _int, _i64, _i64, _vp, _sz, _vp]
_lib.cb_packed_gemm.argtypes = [_vp, _i64, _WP, _vp, _i64, _int, _i64, _int, _int, _int, _vp]
_lib.cb_packed_gemm_scratch.argtypes = [_vp, _i64, _WP, _vp, _i64, _int, _i64, _int, _int, _int, _vp, _sz, _vp]
_lib.cb_packed_gemm_scratch.restype = _int
_lib.cb_gemm_scratch_bytes.argtypes = [_i64, _i64, _i64]
_lib.cb_gemm_scratch_bytes.restype = _sz
_COUNTER_BYTES = 65536 * 4      # the decode kernels' arrival counters at the head of a stream's scratch buffer
_lib.cb_unpack_codes.argtypes = [_vp, _i64, _i64, _int, _vp, _vp]
_lib.cb_max_rho.argtypes = [_int, _int]
_lib.cb_decode_plan.argtypes = [_int, _i64, _i64, _i64, _i64, _i64, _int, ctypes.POINTER(ctypes.c_longlong)]
_lib.cb_set_option.argtypes = [_int, _int]
_lib.cb_set_option.restype = None
_lib.cb_decode_status.argtypes = [ctypes.POINTER(_int)]
for _f in ("cb_packed_gemv", "cb_fused_gate_up", "cb_fused_qkv", "cb_packed_gemm", "cb_unpack_codes",
           "cb_sm_count", "cb_tile_n", "cb_max_rho", "cb_decode_status"):
    getattr(_lib, _f).restype = _int

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_KIND = {"gemv": 0, "qkv": 1, "gate_up": 2}


def _fail(msg: str):
    raise RuntimeError(msg)


def _rc(code: int):
    if code != 0:
        raise RuntimeError(_lib.cb_last_error().decode() or f"libcrispybits_b200 error {code}")


def _ptr(t) -> int:
    return 0 if t is None or t.numel() == 0 else t.data_ptr()


def _check_x(x: torch.Tensor, k: int):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _fail("x must be a CUDA tensor (this build has no CPU path)")
    if x.dim() != 2:
        _fail("x must be [B, K]")
    if not x.is_contiguous():
        _fail("x must be contiguous")
    if x.shape[1] != k:
        _fail("x K != in_features")
    if x.dtype not in _DTYPE:
        _fail("x must be fp16/bf16/fp32")


def _check_weight(x, packed, scales, zeros, bits: int, k: int, gs: int, name: str):
    if not (packed.is_cuda and scales.is_cuda and zeros.is_cuda):
        _fail(f"{name}: tensors must be CUDA")
    if packed.device != x.device or scales.device != x.device or zeros.device != x.device:
        _fail(f"{name}: weight and activation on different devices")
    if packed.dtype != torch.int32:
        _fail(f"{name}: packed must be torch.int32")
    if packed.dim() != 2 or scales.dim() != 2:
        _fail(f"{name}: packed/scales must be 2-D")
    if not (packed.is_contiguous() and scales.is_contiguous() and zeros.is_contiguous()):
        _fail(f"{name}: weight tensors must be contiguous")
    if scales.shape != zeros.shape:
        _fail(f"{name}: scale/zero shape mismatch")
    if scales.shape[0] != packed.shape[0]:
        _fail(f"{name}: metadata rows != output rows")
    if scales.dtype != x.dtype or zeros.dtype != x.dtype:
        _fail(f"{name}: metadata dtype must match x")
    if bits not in (2, 3, 4):
        _fail(f"{name}: bits must be 2/3/4")
    if gs <= 0 or gs % 32:
        _fail(f"{name}: group_size must be a positive multiple of 32")
    if packed.shape[1] != -(-k // 32) * bits:
        _fail(f"{name}: packed row must hold exactly ceil(K/32)*bits words (rows padded to 32 codes)")
    if scales.shape[1] != -(-k // gs):
        _fail(f"{name}: expected ceil(K/group_size) groups")
    align = 16 if bits == 4 else (8 if bits == 2 else 4)
    if packed.data_ptr() % align:
        _fail(f"{name}: packed storage must be {align}-byte aligned for vector loads")


def _bias_or_none(bias, x, n: int):
    if bias is None or bias.numel() == 0:
        return None
    if not bias.is_cuda or bias.device != x.device:
        _fail("bias must be on x's device")
    if bias.numel() != n:
        _fail("bias length must equal out_features")
    if bias.dtype != x.dtype:
        _fail("bias dtype must match x")
    if not bias.is_contiguous():
        _fail("bias must be contiguous")
    return bias


def _check_workspace(ws, x):
    """The reference's 2-int job-queue workspace (host_utils.h:38-47).  The B200 kernels partition work
    statically and need no queue; a caller-supplied workspace is validated and left untouched, so it
    still reads [0, 0] afterwards."""
    if ws is None or ws.numel() < 2:
        return
    if not ws.is_cuda or ws.device != x.device:
        _fail("workspace must be on x's device")
    if ws.dtype != torch.int32 or not ws.is_contiguous():
        _fail("workspace must be contiguous int32")


def _weight(packed, scales, zeros, bias) -> _Weight:
    return _Weight(packed.data_ptr(), scales.data_ptr(), zeros.data_ptr(), _ptr(bias), packed.shape[0])


# Weights that passed their checks, so that a model's repeated calls with the same tensors do not pay for them again:
# (identities of the four tensors, bits, K, group size, activation dtype and device) -> (weak reference to `packed`,
# the record handed to the library).  An identity can be reused after a tensor dies, hence the weak reference; a tensor
# whose storage is swapped in place (`.data = ...`) changes its data pointer, so the four pointers are compared too.
_checked: Dict[tuple, tuple] = {}


def _checked_weight(x, packed, scales, zeros, bias, bits: int, k: int, gs: int, name: str) -> _Weight:
    key = (id(packed), id(scales), id(zeros), id(bias), bits, k, gs, x.dtype, x.device)
    hit = _checked.get(key)
    if hit is not None and hit[0]() is packed:
        w = hit[1]
        if (w.packed == packed.data_ptr() and w.scales == scales.data_ptr() and w.zeros == zeros.data_ptr()
                and (w.bias or 0) == _ptr(bias)):
            return w
    _check_weight(x, packed, scales, zeros, bits, k, gs, name)
    w = _weight(packed, scales, zeros, _bias_or_none(bias, x, packed.shape[0]))
    if len(_checked) >= 8192:
        _checked.clear()
    _checked[key] = (weakref.ref(packed), w)
    return w


_COUNTER_REGION = 65536 * 4      # cb_gemv_scratch_bytes: a fixed region of arrival counters, then split_k * B * V floats


# Split-K scratch: one zero-initialised buffer per (device, stream), grown on demand and kept alive
# for the life of the process (CUDA graphs that captured its address stay valid).  The kernels reset
# the counters they use, so the buffer is zeroed only when it is created.
_scratch: Dict[Tuple[int, int], torch.Tensor] = {}
_retired: List[torch.Tensor] = []


def _scratch_for(x: torch.Tensor, stream: int, nbytes: int):
    if nbytes == 0:
        return None
    key = (x.device.index, stream)
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        if buf is not None:
            _retired.append(buf)   # a captured graph may still point at it
        buf = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=x.device)
        _scratch[key] = buf
    return buf


def _decode_scratch(x, stream: int, B: int, V: int, pk: int):
    """Scratch for a decode call.  Sized for the requested split and, so that the streamlined kernel may
    raise the split when its shared-memory budget asks for it, for at least a 4-way split (the arithmetic of
    cb_gemv_scratch_bytes, done here to save two library calls per launch)."""
    return _scratch_for(x, stream, _COUNTER_REGION + max(pk, 4) * B * V * 4)


class _on_device:
    """`with torch.cuda.device(...)` only when the tensor's device is not the current one."""
    __slots__ = ("ctx",)

    def __init__(self, device):
        self.ctx = None if device.index is None or torch.cuda.current_device() == device.index else torch.cuda.device(device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            return self.ctx.__exit__(*exc)
        return False


def _stream(x) -> int:
    return torch.cuda.current_stream(x.device).cuda_stream


def packed_gemv(x, packed, scales, zeros, bias, bits, in_features, group_size, split_k, rho, act, workspace):
    bits, k, gs, split_k, rho, act = int(bits), int(in_features), int(group_size), int(split_k), int(rho), int(act)
    _check_x(x, k)
    w = _checked_weight(x, packed, scales, zeros, bias, bits, k, gs, "packed_gemv")
    if split_k < 1:
        _fail("split_k must be >= 1")
    if not 0 <= act <= 2:
        _fail("act must be 0 (none), 1 (relu) or 2 (silu)")
    _check_workspace(workspace, x)
    B, n = x.shape[0], packed.shape[0]
    out = torch.empty((B, n), dtype=x.dtype, device=x.device)
    if B == 0:
        return out
    with _on_device(x.device):
        st = _stream(x)
        pk = max(1, min(split_k, -(-k // 32)))
        sc = _decode_scratch(x, st, B, n, pk)
        _rc(_lib.cb_packed_gemv(x.data_ptr(), B, ctypes.byref(w), out.data_ptr(), k, bits, gs, _DTYPE[x.dtype],
                                pk, rho, act, _ptr(sc), 0 if sc is None else sc.numel(), st))
    return out


def packed_gemm(x, packed, scales, zeros, bias, bits, in_features, group_size, act, use_tensor_cores):
    bits, k, gs, act = int(bits), int(in_features), int(group_size), int(act)
    _check_x(x, k)
    _check_weight(x, packed, scales, zeros, bits, k, gs, "packed_gemm")
    if not 0 <= act <= 2:
        _fail("act must be 0 (none), 1 (relu) or 2 (silu)")
    bias = _bias_or_none(bias, x, packed.shape[0])
    M, n = x.shape[0], packed.shape[0]
    out = torch.empty((M, n), dtype=x.dtype, device=x.device)
    if M == 0:
        return out
    with torch.cuda.device(x.device):
        w = _weight(packed, scales, zeros, bias)
        st = _stream(x)
        # scratch for a K split of few-token calls: behind the decode kernels' counter region of the stream's buffer
        need = _lib.cb_gemm_scratch_bytes(M, n, k) if use_tensor_cores else 0
        sc = _scratch_for(x, st, _COUNTER_BYTES + need) if need else None
        _rc(_lib.cb_packed_gemm_scratch(x.data_ptr(), M, ctypes.byref(w), out.data_ptr(), k, bits, gs, _DTYPE[x.dtype],
                                        act, 1 if use_tensor_cores else 0,
                                        0 if sc is None else sc.data_ptr() + _COUNTER_BYTES, need, st))
    return out


def fused_gate_up(x, wg, sg, zg, wu, su, zu, bits, in_features, group_size, split_k, rho, workspace):
    bits, k, gs, split_k, rho = int(bits), int(in_features), int(group_size), int(split_k), int(rho)
    _check_x(x, k)
    _check_weight(x, wg, sg, zg, bits, k, gs, "fused_gate_up(gate)")
    _check_weight(x, wu, su, zu, bits, k, gs, "fused_gate_up(up)")
    if wg.shape != wu.shape:
        _fail("gate/up packed shapes must match")
    if split_k < 1:
        _fail("split_k must be >= 1")
    _check_workspace(workspace, x)
    B, n = x.shape[0], wg.shape[0]
    out = torch.empty((B, n), dtype=x.dtype, device=x.device)
    if B == 0:
        return out
    with torch.cuda.device(x.device):
        st = _stream(x)
        pk = max(1, min(split_k, -(-k // 32)))
        sc = _decode_scratch(x, st, B, 2 * n, pk)
        g, u = _weight(wg, sg, zg, None), _weight(wu, su, zu, None)
        _rc(_lib.cb_fused_gate_up(x.data_ptr(), B, ctypes.byref(g), ctypes.byref(u), out.data_ptr(), k, bits, gs,
                                  _DTYPE[x.dtype], pk, rho, _ptr(sc), 0 if sc is None else sc.numel(), st))
    return out


def fused_qkv(x, wq, sq, zq, bq, wk, sk, zk, bk, wv, sv, zv, bv, rope_cos, rope_sin, head_dim, perm_hd,
              bits, in_features, group_size, split_k, rho, workspace):
    bits, k, gs, split_k, rho = int(bits), int(in_features), int(group_size), int(split_k), int(rho)
    head_dim, perm_hd = int(head_dim), int(perm_hd)
    _check_x(x, k)
    _check_weight(x, wq, sq, zq, bits, k, gs, "fused_qkv(q)")
    _check_weight(x, wk, sk, zk, bits, k, gs, "fused_qkv(k)")
    _check_weight(x, wv, sv, zv, bits, k, gs, "fused_qkv(v)")
    if split_k < 1:
        _fail("split_k must be >= 1")
    B = x.shape[0]
    if perm_hd > 0:
        if perm_hd % 2:
            _fail("perm head_dim must be even")
        if wq.shape[0] % perm_hd or wk.shape[0] % perm_hd:
            _fail("Q/K widths must be multiples of head_dim")
    rope = rope_cos is not None and rope_cos.numel() > 0
    rc = rs = None
    if rope:
        if not (perm_hd > 0 and perm_hd == head_dim):
            _fail("fused RoPE needs Q/K weights stored pair-interleaved with the same head_dim "
                  "(ops.permute_for_rope / install_bitmap(fuse_rope=True))")
        if rope_cos.shape != rope_sin.shape:
            _fail("cos/sin shape mismatch")
        if rope_cos.numel() != B * head_dim:
            _fail("cos/sin must be [B, head_dim] (one row per x row)")
        rc = rope_cos.to(device=x.device, dtype=torch.float32).contiguous()
        rs = rope_sin.to(device=x.device, dtype=torch.float32).contiguous()
    bq, bk, bv = (_bias_or_none(b, x, w.shape[0]) for b, w in ((bq, wq), (bk, wk), (bv, wv)))
    _check_workspace(workspace, x)
    outs = [torch.empty((B, w.shape[0]), dtype=x.dtype, device=x.device) for w in (wq, wk, wv)]
    if B == 0:
        return outs
    with torch.cuda.device(x.device):
        st = _stream(x)
        pk = max(1, min(split_k, -(-k // 32)))
        V = wq.shape[0] + wk.shape[0] + wv.shape[0]
        sc = _decode_scratch(x, st, B, V, pk)
        q, kk, v = _weight(wq, sq, zq, bq), _weight(wk, sk, zk, bk), _weight(wv, sv, zv, bv)
        _rc(_lib.cb_fused_qkv(x.data_ptr(), B, ctypes.byref(q), ctypes.byref(kk), ctypes.byref(v),
                              outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), _ptr(rc), _ptr(rs),
                              head_dim if rope else 0, perm_hd, k, bits, gs, _DTYPE[x.dtype], pk, rho,
                              _ptr(sc), 0 if sc is None else sc.numel(), st))
    return outs


# ------------------------------------------------------------------ column-parallel stacks (no reference counterpart)
class _Scatter(ctypes.Structure):
    """struct cb_scatter of include/crispybits_b200.h"""
    _fields_ = [("peer_out", _vp * 8), ("world", _int), ("n_gather", _i64), ("ld", _i64), ("col", _i64),
                ("sync", _int), ("rank", _int), ("peer_flags", _vp * 8), ("my_flags", _vp), ("epoch", _vp),
                ("done", _vp), ("status", _vp), ("seq", _i64), ("need", _i64)]


class PeerSync:
    """Device words of the in-kernel rank hand-shake (see struct cb_scatter): peer flag arrays, own flag array,
    launch count, CTA counter and status."""

    def __init__(self, peer_flag_ptrs, my_flags: torch.Tensor, epoch: torch.Tensor, done: torch.Tensor,
                 status: torch.Tensor, rank: int, numbered: bool = False):
        self.peer_flag_ptrs, self.rank = list(peer_flag_ptrs), int(rank)
        self.my_flags, self.epoch, self.done, self.status = my_flags, epoch, done, status
        self.numbered = bool(numbered)     # the numbered hand-shake (cb_scatter.sync == 2): seq per launch, publish, step end


_SP = ctypes.POINTER(_Scatter)
_lib.cb_packed_gemv_scatter.argtypes = [_vp, _i64, _WP, _vp, _SP, _i64, _int, _i64, _int, _i64, _i64, _int, _vp, _sz, _vp]
_lib.cb_fused_gate_up_scatter.argtypes = [_vp, _i64, _WP, _WP, _vp, _SP, _i64, _int, _i64, _int, _i64, _i64, _vp, _sz, _vp]
_lib.cb_peer_barrier.argtypes = [ctypes.POINTER(_vp), _vp, _vp, _vp, _int, _int, _vp]
_lib.cb_peer_wait.argtypes = [_SP, _vp]
_lib.cb_peer_publish.argtypes = [_SP, _vp]
_lib.cb_peer_step_end.argtypes = [_SP, _i64, _vp]
for _f in ("cb_packed_gemv_scatter", "cb_fused_gate_up_scatter", "cb_peer_barrier", "cb_peer_wait", "cb_peer_publish",
           "cb_peer_step_end"):
    getattr(_lib, _f).restype = _int


def _scatter(peer_ptrs, n_gather: int, ld: int, col: int, sync: "PeerSync | None" = None, seq: int = 0,
             need: "int | None" = None) -> _Scatter:
    sc = _Scatter()
    for i, ptr in enumerate(peer_ptrs):
        sc.peer_out[i] = ptr
    sc.world, sc.n_gather, sc.ld, sc.col = len(peer_ptrs), n_gather, ld, col
    if sync is not None:
        sc.sync, sc.rank, sc.seq = (2 if sync.numbered else 1), sync.rank, int(seq)
        sc.need = int(seq) if need is None else int(need)
        for i, ptr in enumerate(sync.peer_flag_ptrs):
            sc.peer_flags[i] = ptr
        sc.my_flags, sc.epoch = sync.my_flags.data_ptr(), sync.epoch.data_ptr()
        sc.done, sc.status = sync.done.data_ptr(), sync.status.data_ptr()
    return sc


def packed_gemv_scatter(x, packed, scales, zeros, bias, out, peer_ptrs, n_gather, ld, col, bits, in_features,
                        group_size, split_k, rho, act, sync=None, seq=0, need=None):
    """packed_gemv whose output rows < n_gather go to every rank's gathered buffer (peer pointers) at column
    `col` of a [B, ld] matrix; the other rows go to `out` [B, N].  `seq`: number of the launch within its step, for a
    numbered hand-shake."""
    bits, k, gs, split_k = int(bits), int(in_features), int(group_size), int(split_k)
    _check_x(x, k)
    _check_weight(x, packed, scales, zeros, bits, k, gs, "packed_gemv_scatter")
    bias = _bias_or_none(bias, x, packed.shape[0])
    B, n = x.shape[0], packed.shape[0]
    if out.shape != (B, n) or out.dtype != x.dtype or not out.is_contiguous() or out.device != x.device:
        _fail("packed_gemv_scatter: out must be a contiguous [B, N] tensor of x's dtype on x's device")
    with torch.cuda.device(x.device):
        st = _stream(x)
        pk = max(1, min(split_k, -(-k // 32)))
        sc = _decode_scratch(x, st, B, n, pk)
        w, s = _weight(packed, scales, zeros, bias), _scatter(peer_ptrs, int(n_gather), int(ld), int(col), sync, seq, need)
        _rc(_lib.cb_packed_gemv_scatter(x.data_ptr(), B, ctypes.byref(w), out.data_ptr(), ctypes.byref(s), k, bits, gs,
                                        _DTYPE[x.dtype], pk, int(rho), int(act), _ptr(sc), 0 if sc is None else sc.numel(), st))
    return out


def fused_gate_up_scatter(x, wg, sg, zg, wu, su, zu, out, peer_ptrs, n_gather, ld, col, bits, in_features, group_size,
                          split_k, rho, sync=None, seq=0):
    bits, k, gs, split_k = int(bits), int(in_features), int(group_size), int(split_k)
    _check_x(x, k)
    _check_weight(x, wg, sg, zg, bits, k, gs, "fused_gate_up_scatter(gate)")
    _check_weight(x, wu, su, zu, bits, k, gs, "fused_gate_up_scatter(up)")
    if wg.shape != wu.shape:
        _fail("gate/up packed shapes must match")
    B, n = x.shape[0], wg.shape[0]
    if out.shape != (B, n) or out.dtype != x.dtype or not out.is_contiguous():
        _fail("fused_gate_up_scatter: out must be a contiguous [B, N] tensor of x's dtype")
    with torch.cuda.device(x.device):
        st = _stream(x)
        pk = max(1, min(split_k, -(-k // 32)))
        sc = _decode_scratch(x, st, B, 2 * n, pk)
        g, u, s = _weight(wg, sg, zg, None), _weight(wu, su, zu, None), _scatter(peer_ptrs, int(n_gather), int(ld), int(col), sync, seq)
        _rc(_lib.cb_fused_gate_up_scatter(x.data_ptr(), B, ctypes.byref(g), ctypes.byref(u), out.data_ptr(), ctypes.byref(s),
                                          k, bits, gs, _DTYPE[x.dtype], pk, int(rho), _ptr(sc), 0 if sc is None else sc.numel(), st))
    return out


def peer_barrier(peer_flag_ptrs, my_flags: torch.Tensor, epoch: torch.Tensor, status: torch.Tensor, rank: int):
    """Launch the rank-to-rank barrier kernel on the current stream of my_flags' device."""
    world = len(peer_flag_ptrs)
    arr = (_vp * world)(*peer_flag_ptrs)
    with torch.cuda.device(my_flags.device):
        _rc(_lib.cb_peer_barrier(arr, my_flags.data_ptr(), epoch.data_ptr(), status.data_ptr(), world, int(rank),
                                 torch.cuda.current_stream(my_flags.device).cuda_stream))


def peer_publish(sync: "PeerSync", seq: int):
    """Numbered hand-shake: after scatter launch `seq` of a step, the one-CTA kernel that tells every rank it is done."""
    sc = _scatter([0] * len(sync.peer_flag_ptrs), 0, 1, 0, sync, seq)
    with _on_device(sync.my_flags.device):
        _rc(_lib.cb_peer_publish(ctypes.byref(sc), torch.cuda.current_stream(sync.my_flags.device).cuda_stream))


def peer_step_end(sync: "PeerSync", launches: int):
    """Numbered hand-shake: end of a step of `launches` launches (bounded wait for every rank, then the step base moves)."""
    sc = _scatter([0] * len(sync.peer_flag_ptrs), 0, 1, 0, sync)
    with _on_device(sync.my_flags.device):
        _rc(_lib.cb_peer_step_end(ctypes.byref(sc), int(launches), torch.cuda.current_stream(sync.my_flags.device).cuda_stream))


def peer_wait(sync: "PeerSync"):
    """Launch the bounded wait for the peers' latest hand-shake launch on the current stream."""
    sc = _scatter([0] * len(sync.peer_flag_ptrs), 0, 1, 0, sync)
    with torch.cuda.device(sync.my_flags.device):
        _rc(_lib.cb_peer_wait(ctypes.byref(sc), torch.cuda.current_stream(sync.my_flags.device).cuda_stream))


def unpack_codes(packed: torch.Tensor, bits: int, in_features: int) -> torch.Tensor:
    """int32 codes [N, K] from packed words, computed on the GPU (checked bit-for-bit in the tests)."""
    if not packed.is_cuda or packed.dtype != torch.int32 or packed.dim() != 2 or not packed.is_contiguous():
        _fail("packed must be a contiguous 2-D CUDA int32 tensor")
    k = int(in_features)
    if packed.shape[1] != -(-k // 32) * int(bits):
        _fail("packed row must hold exactly ceil(K/32)*bits words")
    out = torch.empty((packed.shape[0], k), dtype=torch.int32, device=packed.device)
    with torch.cuda.device(packed.device):
        _rc(_lib.cb_unpack_codes(packed.data_ptr(), packed.shape[0], k, int(bits), out.data_ptr(),
                                 torch.cuda.current_stream(packed.device).cuda_stream))
    return out


_lib.cb_fused_gate_up_gemm.argtypes = [_vp, _i64, _WP, _WP, _vp, _i64, _int, _i64, _int, _vp]
_lib.cb_fused_gate_up_gemm.restype = _int


def fused_gate_up_gemm(x, wg, sg, zg, wu, su, zu, bits, in_features, group_size):
    """silu(x Wg^T) * (x Wu^T) for a prefill batch in one launch, or None when the shape is outside the fused
    kernel's domain (the caller then runs two GEMMs and a product, as the reference does)."""
    bits, k, gs = int(bits), int(in_features), int(group_size)
    _check_x(x, k)
    _check_weight(x, wg, sg, zg, bits, k, gs, "fused_gate_up_gemm(gate)")
    _check_weight(x, wu, su, zu, bits, k, gs, "fused_gate_up_gemm(up)")
    if wg.shape != wu.shape:
        _fail("gate/up packed shapes must match")
    if x.dtype not in (torch.float16, torch.bfloat16) or k % 128 or gs % 64:
        return None
    M, n = x.shape[0], wg.shape[0]
    out = torch.empty((M, n), dtype=x.dtype, device=x.device)
    if M == 0:
        return out
    with torch.cuda.device(x.device):
        g, u = _weight(wg, sg, zg, None), _weight(wu, su, zu, None)
        rc = _lib.cb_fused_gate_up_gemm(x.data_ptr(), M, ctypes.byref(g), ctypes.byref(u), out.data_ptr(), k, bits, gs,
                                        _DTYPE[x.dtype], _stream(x))
    if rc == 3:          # CB_ERR_UNSUPPORTED
        return None
    _rc(rc)
    return out


_lib.cb_fused_qkv_gemm.argtypes = [_vp, _i64, _WP, _WP, _WP, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _int, _i64, _int, _vp]
_lib.cb_fused_qkv_gemm.restype = _int


def fused_qkv_gemm(x, wq, sq, zq, bq, wk, sk, zk, bk, wv, sv, zv, bv, rope_cos, rope_sin, head_dim, perm_hd,
                   bits, in_features, group_size):
    """Q, K, V of a prefill batch (+ bias, + RoPE on Q and K, outputs in the original column order) in one launch,
    or None when the shape is outside the fused kernel's domain (every projection's rows a multiple of 128); the
    caller then runs three GEMMs and rotates afterwards, as the reference does."""
    bits, k, gs = int(bits), int(in_features), int(group_size)
    head_dim, perm_hd = int(head_dim), int(perm_hd)
    _check_x(x, k)
    _check_weight(x, wq, sq, zq, bits, k, gs, "fused_qkv_gemm(q)")
    _check_weight(x, wk, sk, zk, bits, k, gs, "fused_qkv_gemm(k)")
    _check_weight(x, wv, sv, zv, bits, k, gs, "fused_qkv_gemm(v)")
    if x.dtype not in (torch.float16, torch.bfloat16) or k % 128 or gs % 64:
        return None
    if any(w.shape[0] % 128 for w in (wq, wk, wv)):
        return None
    M = x.shape[0]
    if perm_hd > 0:
        if perm_hd % 2:
            _fail("perm head_dim must be even")
        if wq.shape[0] % perm_hd or wk.shape[0] % perm_hd:
            _fail("Q/K widths must be multiples of head_dim")
    rope = rope_cos is not None and rope_cos.numel() > 0
    rc = rs = None
    if rope:
        if not (perm_hd > 0 and perm_hd == head_dim):
            _fail("fused RoPE needs Q/K weights stored pair-interleaved with the same head_dim "
                  "(ops.permute_for_rope / install_bitmap(fuse_rope=True))")
        if rope_cos.shape != rope_sin.shape:
            _fail("cos/sin shape mismatch")
        if rope_cos.numel() != M * head_dim:
            _fail("cos/sin must be [M, head_dim] (one row per x row)")
        rc = rope_cos.to(device=x.device, dtype=torch.float32).contiguous()
        rs = rope_sin.to(device=x.device, dtype=torch.float32).contiguous()
    bq, bk, bv = (_bias_or_none(b, x, w.shape[0]) for b, w in ((bq, wq), (bk, wk), (bv, wv)))
    outs = [torch.empty((M, w.shape[0]), dtype=x.dtype, device=x.device) for w in (wq, wk, wv)]
    if M == 0:
        return outs
    with torch.cuda.device(x.device):
        q, kk, v = _weight(wq, sq, zq, bq), _weight(wk, sk, zk, bk), _weight(wv, sv, zv, bv)
        code = _lib.cb_fused_qkv_gemm(x.data_ptr(), M, ctypes.byref(q), ctypes.byref(kk), ctypes.byref(v),
                                      outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), _ptr(rc), _ptr(rs),
                                      head_dim, perm_hd, k, bits, gs, _DTYPE[x.dtype], _stream(x))
    if code == 3:        # CB_ERR_UNSUPPORTED
        return None
    _rc(code)
    return outs


_lib.cb_quantize_pack.argtypes = [_vp, _int, _i64, _i64, _int, _i64, _vp, _vp, _vp, _int, _vp]
_lib.cb_quantize_pack.restype = _int


def quantize_pack(w: torch.Tensor, bits: int, group_size: int, meta_dtype=torch.float16):
    """(packed int32 [N, ceil(K/32)*bits], scales, zeros [N, ceil(K/gs)] of meta_dtype) from a CUDA [N, K] float
    matrix, computed by the library's quantise+pack kernel (bit-identical to the reference's CPU packer)."""
    if not w.is_cuda or w.dim() != 2 or w.dtype not in _DTYPE:
        _fail("quantize_pack: w must be a 2-D CUDA tensor of float32, float16 or bfloat16")
    if meta_dtype not in _DTYPE:
        _fail("quantize_pack: scales/zeros dtype must be float32, float16 or bfloat16")
    bits, gs = int(bits), int(group_size)
    w = w.contiguous()
    n, k = w.shape
    packed = torch.empty((n, -(-k // 32) * bits), dtype=torch.int32, device=w.device)
    scales = torch.empty((n, -(-k // gs)), dtype=meta_dtype, device=w.device)
    zeros = torch.empty_like(scales)
    with torch.cuda.device(w.device):
        _rc(_lib.cb_quantize_pack(w.data_ptr(), _DTYPE[w.dtype], n, k, bits, gs, packed.data_ptr(), scales.data_ptr(),
                                  zeros.data_ptr(), _DTYPE[meta_dtype], torch.cuda.current_stream(w.device).cuda_stream))
    return packed, scales, zeros


def sm_count() -> int:
    n = _lib.cb_sm_count()
    if n < 0:
        _rc(2)
    return int(n)


def tile_n() -> int:
    return int(_lib.cb_tile_n())


def max_rho(bits: int, kind: str = "gemv") -> int:
    if kind not in _KIND:
        _fail("kind must be 'gemv', 'qkv' or 'gate_up'")
    r = _lib.cb_max_rho(int(bits), _KIND[kind])
    if r < 0:
        _rc(1)
    return int(r)


def decode_plan(bits: int, batch: int, rows: int, in_features: int, split_k: int = 1, rho: int = 1, sms: int = 148):
    """Launch plan of the ring decode kernel as a dict (host arithmetic only; no GPU needed), or None when the ring
    kernel does not take the problem."""
    out = (ctypes.c_longlong * 7)()
    if _lib.cb_decode_plan(bits, batch, rows, in_features, split_k, rho, sms, out) != 0:
        return None
    keys = ("grid", "smem_bytes", "split_k", "rows_per_pass", "ring_slots", "passes", "row_slabs")
    return dict(zip(keys, (int(v) for v in out)))


def set_option(option: int, value: int) -> None:
    """0: programmatic dependent launch on/off; 1: force the shape-generic decode kernel (A/B checks)."""
    _lib.cb_set_option(int(option), int(value))


def decode_status() -> int:
    """Synchronise, then read and clear the decode kernels' error word (0 = fine)."""
    out = _int(0)
    _rc(_lib.cb_decode_status(ctypes.byref(out)))
    if out.value:
        _zero_attention_counters(torch.cuda.current_device())
    return int(out.value)


def version() -> str:
    return _lib.cb_version().decode()


# ------------------------------------------------------------------ attention and the 4-bit cache (no reference counterpart)
class _KV4Cache(ctypes.Structure):
    """struct cb_kv4_cache of include/crispybits_b200.h"""
    _fields_ = [("pages", _vp), ("n_pages", _i64), ("kv_heads", _i64), ("head_dim", _int), ("group_size", _int),
                ("page_size", _int), ("dtype", _int)]


_KP = ctypes.POINTER(_KV4Cache)
_lib.cb_kv4_block_bytes.argtypes = [_int, _int]
_lib.cb_kv4_block_bytes.restype = _sz
_lib.cb_kv4_append.argtypes = [_KP, _vp, _vp, ctypes.POINTER(_i64), _i64, _vp, _i64, _i64, _vp, _vp, _vp]
_lib.cb_kv4_read.argtypes = [_KP, _vp, _vp, _i64, _vp, _i64, _i64, _vp, _vp, _vp]
_lib.cb_kv4_attention.argtypes = [_KP, _vp, ctypes.POINTER(_i64), _vp, _i64, _i64, _i64, _vp, _i64, _vp, ctypes.c_float,
                                  _vp, _sz, _vp, _sz, _vp]
_lib.cb_kv4_attention_counters.argtypes = [_i64, _i64, _i64, _i64]
_lib.cb_kv4_attention_counters.restype = _i64
_lib.cb_kv4_attention_partial_bytes.argtypes = [_i64, _i64, _i64, _int]
_lib.cb_kv4_attention_partial_bytes.restype = _sz
for _f in ("cb_kv4_append", "cb_kv4_read", "cb_kv4_attention"):
    getattr(_lib, _f).restype = _int


def kv4_block_bytes(head_dim: int, group_size: int) -> int:
    """Bytes that 16 tokens of one head take in the 4-bit cache; 0: no kernel for this head_dim and group_size."""
    return int(_lib.cb_kv4_block_bytes(int(head_dim), int(group_size)))


def _kv4_record(cache, who: str) -> _KV4Cache:
    """The library's record of a cache.  It is made and checked once, and kept by the cache it describes."""
    pages, rec = cache.pages, cache.__dict__.get("_record")
    if rec is not None and rec.pages == pages.data_ptr():
        return rec
    if not pages.is_cuda or pages.dtype != torch.uint8 or pages.dim() != 3 or not pages.is_contiguous():
        _fail(f"{who}: the cache's pages must be a contiguous 3-D CUDA uint8 tensor")
    if cache.dtype not in (torch.float16, torch.bfloat16):
        _fail(f"{who}: the cache's dtype must be float16 or bfloat16")
    if pages.shape[2] * 16 != cache.page_size * kv4_block_bytes(cache.head_dim, cache.group_size):
        _fail(f"{who}: pages do not fit the cache's head_dim, group_size and page_size")
    if pages.numel() == 0:
        _fail(f"{who}: the cache has no pages")
    rec = _KV4Cache(pages.data_ptr(), pages.shape[0], pages.shape[1], cache.head_dim, cache.group_size, cache.page_size,
                    _DTYPE[cache.dtype])
    cache.__dict__["_record"] = rec
    return rec


# The checks below are written for the call that is in order, which takes a few attribute reads; what is wrong with one that is not is
# said by the function that follows.
def _check_index(t, device: int, n: int, name: str, who: str):
    if getattr(t, "dtype", None) is torch.int32 and t.get_device() == device and t.shape == (n,) and t.is_contiguous():
        return
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_cuda or t.get_device() != device:
        _fail(f"{who}: {name} must be an int32 tensor on the device of the others")
    _fail(f"{who}: {name} must be contiguous of shape [{n}]")


def _check_table(page_table, device: int, who: str):
    if getattr(page_table, "dtype", None) is not torch.int32 or page_table.get_device() != device:
        _fail(f"{who}: page_table must be an int32 tensor on the cache's device")
    if page_table.dim() != 2 or not page_table.is_contiguous():
        _fail(f"{who}: page_table must be contiguous [sequences, pages]")


def _vector_rows(t: torch.Tensor, positive: bool = False):
    """(t, its strides) where every row of the last dimension is contiguous and 16-byte aligned (`positive`: and no
    other stride is 0, as in an expanded tensor), else of a contiguous copy."""
    st = t.stride()
    if st[-1] == 1 and not (t.data_ptr() & 15):
        bits = 0
        for s in st[:-1]:
            bits |= s
        if not bits & 7 and not (positive and 0 in st):
            return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def _empty(like: torch.Tensor) -> torch.Tensor:
    """Contiguous, uninitialised, of the shape, dtype and device of `like` (by the shorter way where there is one)."""
    return torch.empty_like(like) if like.is_contiguous() else torch.empty(like.shape, dtype=like.dtype, device=like.device)


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def kv4_append(cache, k, v, page_table, starts, cu_seqlens):
    """k, v [tokens, kv_heads, head_dim] -> the cache's pages (struct cb_kv4_cache; cb_kv4_append)."""
    rec, dev = _kv4_record(cache, "kv4_append"), cache.pages.get_device()
    want = (rec.kv_heads, rec.head_dim)
    for t, name in ((k, "k"), (v, "v")):
        if t.get_device() != dev or t.dtype is not cache.dtype:
            _fail(f"kv4_append: {name} must be of the cache's dtype, on its device")
        if t.dim() != 3 or t.shape[1:] != want:
            _fail(f"kv4_append: {name} must be [tokens, {rec.kv_heads}, {rec.head_dim}]")
    n = k.shape[0]
    if v.shape[0] != n:
        _fail("kv4_append: k and v must have the same shape")
    _check_table(page_table, dev, "kv4_append")
    seqs, pages = page_table.shape
    _check_index(starts, dev, seqs, "starts", "kv4_append")
    if cu_seqlens is not None:
        _check_index(cu_seqlens, dev, seqs + 1, "cu_seqlens", "kv4_append")
    if n == 0:
        return
    (k, sk), (v, sv) = _vector_rows(k), _vector_rows(v)
    strides = (_i64 * 4)(sk[0], sk[1], sv[0], sv[1])
    with _on_device(k.device):
        _rc(_lib.cb_kv4_append(rec, k.data_ptr(), v.data_ptr(), strides, n, page_table.data_ptr(), pages, seqs, starts.data_ptr(),
                               None if cu_seqlens is None else cu_seqlens.data_ptr(), _raw_stream(dev)))


def kv4_read(cache, page_table, starts, cu_seqlens, n_tokens: int):
    """(k, v) [tokens, kv_heads, head_dim]: the values that the cache holds for the named tokens (cb_kv4_read)."""
    rec, dev = _kv4_record(cache, "kv4_read"), cache.pages.get_device()
    _check_table(page_table, dev, "kv4_read")
    seqs, pages = page_table.shape
    n = int(n_tokens)
    if n < 0:
        _fail("kv4_read: n_tokens must not be negative")
    _check_index(starts, dev, seqs, "starts", "kv4_read")
    if cu_seqlens is not None:
        _check_index(cu_seqlens, dev, seqs + 1, "cu_seqlens", "kv4_read")
    device = cache.pages.device
    k = torch.empty((n, rec.kv_heads, rec.head_dim), dtype=cache.dtype, device=device)
    v = torch.empty_like(k)
    if n:
        with _on_device(device):
            _rc(_lib.cb_kv4_read(rec, k.data_ptr(), v.data_ptr(), n, page_table.data_ptr(), pages, seqs, starts.data_ptr(),
                                 None if cu_seqlens is None else cu_seqlens.data_ptr(), _raw_stream(dev)))
    return k, v


# Scratch of the attention operators.  Eager calls: counters (zeroed when made; every call leaves them zero) and partial
# sums of one (device, stream), where calls run one after another.  Captured calls: partial sums from the graph's own
# pool, and counters that no other call ever gets, cut from a slab zeroed beforehand -- two graphs may then run at the
# same time.  A capture that finds no slab, or an empty one, zeroes its counters inside the graph; eager calls see to it that the next finds one at
# least half full.
_attention_eager: Dict[Tuple[int, int], Tuple[torch.Tensor, torch.Tensor]] = {}
_attention_slab: Dict[int, List] = {}          # device index -> [tensor, next free element]
_attention_spent: List[torch.Tensor] = []      # slabs that graphs count in and nothing more is cut from
_ATTENTION_SLAB = 1 << 18
_attention_lock = threading.Lock()
_prompt_bytes: Dict[Tuple[int, ...], Tuple[int, int]] = {}   # (device index, head_dim, sizes) -> bytes of counters and partial, cb_prompt_attention_scratch_for
_partial_bytes: Dict[Tuple[int, bool, int], int] = {}      # (device index, more than 8 rows, head_dim) -> cb_kv4_attention_partial_bytes


def prepare_attention(device: torch.device):
    """Make the slab of zeroed counters that captured calls on this device draw from (not inside a capture)."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    if index not in _attention_slab and not torch.cuda.is_current_stream_capturing():
        with _attention_lock, _on_device(torch.device("cuda", index)):
            slab = torch.zeros(_ATTENTION_SLAB, dtype=torch.int32, device=torch.device("cuda", index))
            torch.cuda.current_stream(index).synchronize()       # visible to whatever stream a graph will run on
            _attention_slab.setdefault(index, [slab, 0])


def _renew_attention_slab(device, slab: List):
    """Half of the counters for captures are given out: the next captures draw from another slab.  The old one stays, graphs count in it."""
    fresh = torch.zeros(_ATTENTION_SLAB, dtype=torch.int32, device=device)
    torch.cuda.current_stream(device).synchronize()
    with _attention_lock:
        if slab[1] > _ATTENTION_SLAB // 2:
            _attention_spent.append(slab[0])
            slab[0], slab[1] = fresh, 0


def _zero_attention_counters(index: int):
    """A launch that gave up a wait leaves counters that are not zero, and later launches would join parts that are not there.  Any status is taken
    for one: it may hide another."""
    torch.cuda.synchronize(index)
    with _attention_lock, _on_device(torch.device("cuda", index)):
        kept = [have[0] for (dev, _), have in list(_attention_eager.items()) if dev == index]
        slabs = [slab[0] for slab in _attention_slab.values()] + _attention_spent
        for counters in kept + [slab for slab in slabs if slab.get_device() == index]:
            counters.zero_()
    torch.cuda.synchronize(index)


def _attention_scratch(device, dev: int, stream: int, counters: int, nbytes: int):
    if torch.cuda.is_current_stream_capturing():
        partial = torch.empty(nbytes, dtype=torch.uint8, device=device)
        need = -(-counters // 32) * 32
        with _attention_lock:
            slab = _attention_slab.get(dev)
            at = _ATTENTION_SLAB if slab is None else slab[1]
            if at + need <= _ATTENTION_SLAB:
                slab[1] = at + need
        if at + need > _ATTENTION_SLAB:
            return torch.zeros(counters, dtype=torch.int32, device=device), partial
        return slab[0][at:at + need], partial
    slab = _attention_slab.get(dev)
    if slab is not None and slab[1] > _ATTENTION_SLAB // 2:
        _renew_attention_slab(device, slab)
    have = _attention_eager.get((dev, stream))
    if have is None or have[0].numel() < counters or have[1].numel() < nbytes:
        prepare_attention(device)
        counts, partial = have or (None, None)                   # what is large enough stays: other calls may need it as it is
        if counts is None or counts.numel() < counters:
            counts = torch.zeros(max(counters, 8192), dtype=torch.int32, device=device)
        if partial is None or partial.numel() < nbytes:
            partial = torch.empty(nbytes, dtype=torch.uint8, device=device)
        have = _attention_eager[(dev, stream)] = (counts, partial)
    return have


def kv4_attention(q, cache, page_table, lengths, scale: float):
    """q [B, T, H, head_dim] or [B, H, head_dim] -> as q (cb_kv4_attention)."""
    rec, dev = _kv4_record(cache, "kv4_attention"), cache.pages.get_device()
    if q.get_device() != dev or q.dtype is not cache.dtype:
        _fail("kv4_attention: q must be of the cache's dtype, on its device")
    shape, kv, D = q.shape, rec.kv_heads, rec.head_dim
    if len(shape) not in (3, 4) or shape[-1] != D:
        _fail(f"kv4_attention: q must be [B, T, H, {D}] or [B, H, {D}]")
    B, T, H = shape[0], shape[1] if len(shape) == 4 else 1, shape[-2]
    if H % kv:
        _fail("kv4_attention: q's heads must be a multiple of the cache's")
    _check_table(page_table, dev, "kv4_attention")
    if page_table.shape[0] != B:
        _fail("kv4_attention: page_table needs one row for each sequence of q")
    _check_index(lengths, dev, B, "lengths", "kv4_attention")
    device = q.device
    out = _empty(q)
    if B == 0 or T == 0 or H == 0:
        return out
    q, st = _vector_rows(q)
    rows = T * (H // kv)
    counters = B * kv * (1 if rows <= 8 else -(-rows // 16))
    with _on_device(device):
        key = (dev, rows > 8, D)
        nbytes = _partial_bytes.get(key)
        if nbytes is None:
            nbytes = _partial_bytes[key] = _lib.cb_kv4_attention_partial_bytes(T, H, kv, D)
        stream = _raw_stream(dev)
        counts, partial = _attention_scratch(device, dev, stream, counters, nbytes)
        _rc(_lib.cb_kv4_attention(rec, q.data_ptr(), (_i64 * 3)(st[0], st[1] if len(st) == 4 else 0, st[-2]), out.data_ptr(), B, T, H,
                                  page_table.data_ptr(), page_table.shape[1], lengths.data_ptr(), scale,
                                  counts.data_ptr(), counters * 4, partial.data_ptr(), nbytes, stream))
    return out


_lib.cb_prompt_attention.argtypes = [_vp, _vp, _vp, ctypes.POINTER(_i64), _vp, _i64, _i64, _i64, _i64, _int, _int, _vp, _vp, _i64,
                                     ctypes.c_float, _int, _vp, _sz, _vp, _sz, _vp]
_lib.cb_prompt_attention.restype = _int
_lib.cb_prompt_attention_scratch_for.argtypes = [_i64, _i64, _i64, _i64, _int, ctypes.POINTER(_sz)]
_lib.cb_prompt_attention_scratch_for.restype = _sz


def prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k, scale: float, causal: bool, out=None):
    """q [Tq, H, D], k and v [Tk, Hkv, D] -> [Tq, H, D] (cb_prompt_attention)."""
    who = "prompt_attention"
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        _fail(f"{who}: q must be a CUDA tensor (this build has no CPU path)")
    dtype, dev = q.dtype, q.get_device()
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        _fail(f"{who}: q must be float16 or bfloat16")
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        _fail(f"{who}: q must be [Tq, H, head_dim], k and v [Tk, Hkv, head_dim]")
    if k.get_device() != dev or v.get_device() != dev or k.dtype is not dtype or v.dtype is not dtype:
        _fail(f"{who}: q, k and v must be of one dtype, on one device")
    shape = q.shape
    tq, h, d = shape
    tk, hkv, dk = k.shape
    if dk != d or v.shape != k.shape:
        _fail(f"{who}: k and v must have the same shape, with q's head_dim")
    if hkv == 0 or h % hkv:
        _fail(f"{who}: q's heads must be a multiple of k's")
    if not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or len(cu_seqlens) < 1:
        _fail(f"{who}: cu_seqlens must hold the first query of each sequence and their end")
    n = cu_seqlens.shape[0]
    _check_index(cu_seqlens, dev, n, "cu_seqlens", who)
    if cu_seqlens_k is not cu_seqlens:
        _check_index(cu_seqlens_k, dev, n, "cu_seqlens_k", who)
    device = q.device
    if out is None:
        out = _empty(q)
    elif out.shape != shape or out.dtype != dtype or out.device != device or not out.is_contiguous() or out.data_ptr() % 16:
        _fail(f"{who}: out must be contiguous and 16-byte aligned, of q's shape, dtype and device")
    if tq == 0 or h == 0 or n == 1:
        return out
    (q, sq), (k, sk), (v, sv) = _vector_rows(q, True), _vector_rows(k, True), _vector_rows(v, True)
    strides = (_i64 * 6)(sq[0], sq[1], sk[0], sk[1], sv[0], sv[1])
    with _on_device(device):
        key = (dev, d, tq, tk, h, n)
        stream, sizes = _raw_stream(dev), _prompt_bytes.get(key)
        if sizes is None:
            if len(_prompt_bytes) > 4096:
                _prompt_bytes.clear()
            cbytes = _sz(0)
            nbytes = _lib.cb_prompt_attention_scratch_for(tq, tk, h, n - 1, d, cbytes)
            sizes = _prompt_bytes[key] = (max(cbytes.value, 4), max(nbytes, 16))
        counts, partial = _attention_scratch(device, dev, stream, sizes[0] // 4, sizes[1])
        _rc(_lib.cb_prompt_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, out.data_ptr(), tq, tk, h, hkv, d,
                                     _DTYPE[dtype], cu_seqlens.data_ptr(), cu_seqlens_k.data_ptr(), n - 1, scale,
                                     1 if causal else 0, counts.data_ptr(), sizes[0], partial.data_ptr(), sizes[1], stream))
    return out
