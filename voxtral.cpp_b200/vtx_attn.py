"""Host-side mirror of ggml_flash_attn_ext over the libvtx_fa.so C ABI.

This is the Python face of the node voxtral.cpp builds at src/voxtral.cpp:1611
(encoder) and src/voxtral.cpp:1802 (decoder): same operands, same argument
meaning (ggml views [D, n, H, B] -> here torch tensors (B, H, n, D) with any
strides), same result layout (ggml dst [Dv, Hq, n_q, B] -> torch (B, n_q, Hq,
Dv) float32).  Errors from the library raise ``VtxError`` (ggml would abort
with GGML_ASSERT).  torch supplies device memory and streams only; all
arithmetic runs in the library's sm_100a kernels.  There is no CPU fallback:
without the library or an sm_100 device every call raises.
"""
from __future__ import annotations

import ctypes
import os
import threading
from typing import Optional, Sequence

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libvtx_fa.so")

F32, F16, Q8_0 = 0, 1, 8
QK8_0, Q8_0_BLOCK = 32, 34

STATUS = {0: "ok", -1: "null pointer", -2: "type", -3: "shape", -4: "stride", -5: "unsupported",
          -6: "workspace", -7: "cuda", -8: "no sm_100 device"}


class VtxError(RuntimeError):
    def __init__(self, status: int, what: str = ""):
        self.status = status
        super().__init__(f"vtx status {status} ({STATUS.get(status, '?')}){': ' + what if what else ''}")


class VtxTensor(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("reserved", ctypes.c_int32),
                ("ne", ctypes.c_int64 * 4), ("nb", ctypes.c_size_t * 4),
                ("data", ctypes.c_void_p)]


class FaParams(ctypes.Structure):
    _fields_ = [("scale", ctypes.c_float), ("max_bias", ctypes.c_float),
                ("logit_softcap", ctypes.c_float), ("causal", ctypes.c_int32),
                ("window", ctypes.c_int32), ("reserved", ctypes.c_int32 * 3)]


class DecodeBatch(ctypes.Structure):
    _fields_ = [("n_seq", ctypes.c_int32), ("n_head_q", ctypes.c_int32),
                ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("kv_type", ctypes.c_int32), ("max_kv_len", ctypes.c_int32),
                ("kv_nb1", ctypes.c_size_t), ("kv_nb2", ctypes.c_size_t),
                ("q", ctypes.c_void_p), ("k_ptrs", ctypes.c_void_p),
                ("v_ptrs", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("dst", ctypes.c_void_p), ("scale", ctypes.c_float),
                ("reserved", ctypes.c_int32), ("fresh_row", ctypes.c_void_p)]


class KvAppendArgs(ctypes.Structure):
    """vtx_kv_append_args (include/vtx_fa.h)."""
    _fields_ = [("n_tokens", ctypes.c_int32), ("n_head_q", ctypes.c_int32),
                ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("kv_type", ctypes.c_int32), ("freq_base", ctypes.c_float),
                ("q", ctypes.c_void_p), ("q_nb1", ctypes.c_size_t),
                ("q_out", ctypes.c_void_p), ("q_out_nb1", ctypes.c_size_t),
                ("k", ctypes.c_void_p), ("k_nb1", ctypes.c_size_t),
                ("v", ctypes.c_void_p), ("v_nb1", ctypes.c_size_t),
                ("positions", ctypes.c_void_p), ("slots", ctypes.c_void_p),
                ("k_cache", ctypes.c_void_p), ("v_cache", ctypes.c_void_p),
                ("k_cache_ptrs", ctypes.c_void_p), ("v_cache_ptrs", ctypes.c_void_p),
                ("cache_nb1", ctypes.c_size_t), ("reserved", ctypes.c_int32 * 4)]


class DecodeLayerArgs(ctypes.Structure):
    """vtx_decode_layer_args (include/vtx_fa.h)."""
    _fields_ = [("n_seq", ctypes.c_int32), ("n_head_q", ctypes.c_int32),
                ("n_head_kv", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("kv_type", ctypes.c_int32), ("max_kv_len", ctypes.c_int32),
                ("freq_base", ctypes.c_float), ("scale", ctypes.c_float),
                ("q", ctypes.c_void_p), ("q_nb1", ctypes.c_size_t),
                ("k", ctypes.c_void_p), ("k_nb1", ctypes.c_size_t),
                ("v", ctypes.c_void_p), ("v_nb1", ctypes.c_size_t),
                ("positions", ctypes.c_void_p), ("slots", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("k_cache_ptrs", ctypes.c_void_p), ("v_cache_ptrs", ctypes.c_void_p),
                ("cache_nb1", ctypes.c_size_t), ("dst", ctypes.c_void_p), ("dst_nb1", ctypes.c_size_t),
                ("early", ctypes.c_int32), ("reserved", ctypes.c_int32 * 3)]


class OutProjArgs(ctypes.Structure):
    """vtx_out_proj_args (include/vtx_fa.h)."""
    _fields_ = [("attn", ctypes.c_void_p), ("head_block", ctypes.c_int32), ("reserved", ctypes.c_int32),
                ("block_nb", ctypes.c_size_t), ("w", ctypes.c_void_p), ("bias", ctypes.c_void_p),
                ("residual", ctypes.c_void_p), ("dst", ctypes.c_void_p)]


class VtxPagedKv(ctypes.Structure):
    """vtx_paged_kv (include/vtx_fa.h)."""
    _fields_ = [("k", VtxTensor), ("v", VtxTensor), ("page_table", ctypes.c_void_p), ("kv_len", ctypes.c_void_p),
                ("q_start", ctypes.c_void_p), ("n_seq", ctypes.c_int32), ("max_pages", ctypes.c_int32),
                ("n_tokens", ctypes.c_int32), ("max_new", ctypes.c_int32), ("max_kv_len", ctypes.c_int32),
                ("reserved", ctypes.c_int32)]


class KvAppendPagedArgs(ctypes.Structure):
    """vtx_kv_append_paged_args (include/vtx_fa.h)."""
    _fields_ = [("kv", ctypes.c_void_p), ("n_head_q", ctypes.c_int32), ("q_out_type", ctypes.c_int32),
                ("freq_base", ctypes.c_float), ("row_cap", ctypes.c_int32),
                ("q", ctypes.c_void_p), ("q_nb1", ctypes.c_size_t),
                ("q_out", ctypes.c_void_p), ("q_out_nb1", ctypes.c_size_t),
                ("k", ctypes.c_void_p), ("k_nb1", ctypes.c_size_t),
                ("v", ctypes.c_void_p), ("v_nb1", ctypes.c_size_t),
                ("positions", ctypes.c_void_p), ("row_pos", ctypes.c_void_p), ("score", ctypes.c_void_p)]


class FlashAttnPagedArgs(ctypes.Structure):
    """vtx_flash_attn_paged_args (include/vtx_fa.h)."""
    _fields_ = [("kv", ctypes.c_void_p), ("q", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("lse", ctypes.c_void_p),
                ("params", ctypes.c_void_p)]


class KvScorePagedArgs(ctypes.Structure):
    """vtx_kv_score_paged_args (include/vtx_fa.h)."""
    _fields_ = [("kv", ctypes.c_void_p), ("q", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("params", ctypes.c_void_p),
                ("score", ctypes.c_void_p), ("score_out", ctypes.c_void_p), ("row_cap", ctypes.c_int32),
                ("observe", ctypes.c_int32), ("decay", ctypes.c_float), ("reserved", ctypes.c_int32)]


class KvEvictPagedArgs(ctypes.Structure):
    """vtx_kv_evict_paged_args (include/vtx_fa.h)."""
    _fields_ = [("kv", ctypes.c_void_p), ("score", ctypes.c_void_p), ("row_pos", ctypes.c_void_p),
                ("next_pos", ctypes.c_void_p), ("score_out", ctypes.c_void_p), ("pos_out", ctypes.c_void_p),
                ("src_out", ctypes.c_void_p), ("kv_len_out", ctypes.c_void_p), ("keep", ctypes.c_int32),
                ("n_sink", ctypes.c_int32), ("n_recent", ctypes.c_int32), ("row_cap", ctypes.c_int32),
                ("out_cap", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class EncChunk(ctypes.Structure):
    """vtx_enc_chunk (include/vtx_fa.h): one chunk of the realtime encoder run."""
    _fields_ = [("mel_offset", ctypes.c_int32), ("mel_frames", ctypes.c_int32), ("n_tokens", ctypes.c_int32),
                ("skip", ctypes.c_int32), ("stride", ctypes.c_int32), ("rope_offset", ctypes.c_int32),
                ("write_offset", ctypes.c_int32), ("reserved", ctypes.c_int32)]

    def as_dict(self) -> dict:
        return {f: getattr(self, f) for f, _ in self._fields_ if f != "reserved"}


_lib = None


def load(path: str = LIB_PATH):
    """Load libvtx_fa.so (built by build.py).  Raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise RuntimeError(f"libvtx_fa.so not built ({path}); run voxtral.cpp_b200/build.py")
    L = ctypes.CDLL(path)
    P = ctypes.POINTER
    L.vtx_flash_attn_ext.argtypes = [P(VtxTensor), P(VtxTensor), P(VtxTensor), P(VtxTensor),
                                     P(FaParams), P(VtxTensor), ctypes.c_void_p, ctypes.c_size_t,
                                     ctypes.c_void_p]
    L.vtx_flash_attn_ext.restype = ctypes.c_int
    L.vtx_flash_attn_ext_workspace.argtypes = [P(VtxTensor), P(VtxTensor), P(VtxTensor), P(FaParams)]
    L.vtx_flash_attn_ext_workspace.restype = ctypes.c_size_t
    L.vtx_flash_attn_decode_batched.argtypes = [P(DecodeBatch), ctypes.c_void_p, ctypes.c_size_t,
                                                ctypes.c_void_p]
    L.vtx_flash_attn_decode_batched.restype = ctypes.c_int
    L.vtx_flash_attn_decode_batched_workspace.argtypes = [P(DecodeBatch)]
    L.vtx_flash_attn_decode_batched_workspace.restype = ctypes.c_size_t
    L.vtx_read_device_error.argtypes = [ctypes.c_void_p]
    L.vtx_read_device_error.restype = ctypes.c_int
    L.vtx_strerror.argtypes = [ctypes.c_int]
    L.vtx_strerror.restype = ctypes.c_char_p
    L.vtx_abi_version.argtypes = []
    L.vtx_abi_version.restype = ctypes.c_int
    L.vtx_kv_append.argtypes = [P(KvAppendArgs), ctypes.c_void_p]
    L.vtx_kv_append.restype = ctypes.c_int
    L.vtx_decode_advance.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32,
                                     ctypes.c_int32, ctypes.c_void_p]
    L.vtx_decode_advance.restype = ctypes.c_int
    L.vtx_encoder_chunk_plan.argtypes = [ctypes.c_int32, P(EncChunk), ctypes.c_int32, P(ctypes.c_int32),
                                         P(ctypes.c_int32)]
    L.vtx_encoder_chunk_plan.restype = ctypes.c_int
    L.vtx_encoder_stitch.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_void_p,
                                     ctypes.c_size_t, ctypes.c_size_t, P(EncChunk), ctypes.c_int32,
                                     ctypes.c_void_p]
    L.vtx_encoder_stitch.restype = ctypes.c_int
    L.vtx_attn_out_proj.argtypes = [P(OutProjArgs), ctypes.c_void_p]
    L.vtx_attn_out_proj.restype = ctypes.c_int
    L.vtx_decode_layer.argtypes = [P(DecodeLayerArgs), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    L.vtx_decode_layer.restype = ctypes.c_int
    L.vtx_decode_layer_workspace.argtypes = [P(DecodeLayerArgs)]
    L.vtx_decode_layer_workspace.restype = ctypes.c_size_t
    L.vtx_kv_append_paged.argtypes = [P(KvAppendPagedArgs), ctypes.c_void_p]
    L.vtx_kv_append_paged.restype = ctypes.c_int
    L.vtx_flash_attn_paged_workspace.argtypes = [P(VtxPagedKv), ctypes.c_int32]
    L.vtx_flash_attn_paged_workspace.restype = ctypes.c_size_t
    L.vtx_flash_attn_paged.argtypes = [P(FlashAttnPagedArgs), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    L.vtx_flash_attn_paged.restype = ctypes.c_int
    L.vtx_kv_score_paged.argtypes = [P(KvScorePagedArgs), ctypes.c_void_p]
    L.vtx_kv_score_paged.restype = ctypes.c_int
    L.vtx_kv_evict_paged_workspace.argtypes = [P(VtxPagedKv)]
    L.vtx_kv_evict_paged_workspace.restype = ctypes.c_size_t
    L.vtx_kv_evict_paged.argtypes = [P(KvEvictPagedArgs), ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    L.vtx_kv_evict_paged.restype = ctypes.c_int
    _lib = L
    return L


def _ggml_type(t: torch.Tensor, kv_type: Optional[int]) -> int:
    if kv_type is not None:
        return kv_type
    if t.dtype == torch.float32:
        return F32
    if t.dtype == torch.float16:
        return F16
    raise VtxError(-2, f"dtype {t.dtype}")


def desc(t: Optional[torch.Tensor], ttype: Optional[int] = None) -> Optional[VtxTensor]:
    """ggml descriptor of a torch view: shape (B, H, n, D) -> ne [D, n, H, B].
    Q8_0 tensors are uint8 with the last axis holding D/32 blocks of 34 bytes."""
    if t is None:
        return None
    if t.dim() > 4:
        raise VtxError(-3, "at most 4 dims")
    ttype = _ggml_type(t, ttype)
    shape = [1] * (4 - t.dim()) + list(t.shape)
    es = t.element_size()
    strides = [0] * (4 - t.dim()) + [s * es for s in t.stride()]
    ne = list(reversed(shape))
    nb = list(reversed(strides))
    if ttype == Q8_0:
        ne[0] = ne[0] // Q8_0_BLOCK * QK8_0
        nb[0] = Q8_0_BLOCK
    row = nb[0] * (ne[0] // QK8_0 if ttype == Q8_0 else ne[0])
    for i in range(1, 4):
        if nb[i] == 0 or ne[i] == 1:
            nb[i] = nb[i] or (row if i == 1 else nb[i - 1] * ne[i - 1])
    d = VtxTensor()
    d.type = ttype
    for i in range(4):
        d.ne[i] = ne[i]
        d.nb[i] = nb[i]
    d.data = t.data_ptr()
    return d


def params(scale: float, max_bias: float = 0.0, logit_softcap: float = 0.0,
           causal: bool = False, window: int = 0) -> FaParams:
    p = FaParams()
    p.scale, p.max_bias, p.logit_softcap = float(scale), float(max_bias), float(logit_softcap)
    p.causal, p.window = int(bool(causal)), int(window)
    return p


def _check(rc: int, what: str = "") -> None:
    if rc != 0:
        raise VtxError(rc, what)


def _empty(shape, dtype: torch.dtype, device: torch.device, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """A tensor that a call on `stream` writes.  It comes from that stream's memory:
    a block of the current one's may still be in use by work queued there, which
    `stream` does not wait for.  The current stream counts as a user of it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        t = torch.empty(shape, dtype=dtype, device=device)
    t.record_stream(torch.cuda.current_stream(device))
    return t


def workspace_bytes(q, k, v, scale, max_bias=0.0, logit_softcap=0.0, causal=False, window=0,
                    kv_type=None) -> int:
    L = load()
    p = params(scale, max_bias, logit_softcap, causal, window)
    n = L.vtx_flash_attn_ext_workspace(ctypes.byref(desc(q)), ctypes.byref(desc(k, kv_type)),
                                       ctypes.byref(desc(v, kv_type)), ctypes.byref(p))
    if n == ctypes.c_size_t(-1).value:
        raise VtxError(-3, "operands rejected")
    return int(n)


def flash_attn_ext(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                   mask: Optional[torch.Tensor] = None, scale: float = 1.0,
                   max_bias: float = 0.0, logit_softcap: float = 0.0, *,
                   causal: bool = False, window: int = 0, kv_type: Optional[int] = None,
                   out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """ggml_flash_attn_ext(ctx, q, k, v, mask, scale, max_bias, logit_softcap).

    q: (B, Hq, n_q, D) F32/F16 view; k, v: (B, Hkv, n_kv, D) F16/F32 or Q8_0
    bytes (kv_type=Q8_0); mask: (n_q', n_kv) / (B|1, Hq|1, n_q', n_kv) F16 or
    None.  Returns (B, n_q, Hq, D) float32 (ggml's permuted dst)."""
    L = load()
    B, Hq, n_q = q.shape[0], q.shape[1], q.shape[2]
    Dv = v.shape[-1] if (kv_type or _ggml_type(v, None)) != Q8_0 else v.shape[-1] // Q8_0_BLOCK * QK8_0
    if out is None:
        out = _empty((B, n_q, Hq, Dv), torch.float32, q.device, stream)
    p = params(scale, max_bias, logit_softcap, causal, window)
    dq, dk, dv = desc(q), desc(k, kv_type), desc(v, kv_type)
    need = L.vtx_flash_attn_ext_workspace(ctypes.byref(dq), ctypes.byref(dk), ctypes.byref(dv), ctypes.byref(p))
    if need == ctypes.c_size_t(-1).value:
        raise VtxError(-3, "operands rejected")
    if need and (workspace is None or workspace.numel() * workspace.element_size() < need):
        workspace = _empty((need,), torch.uint8, q.device, stream)
    ws_ptr = workspace.data_ptr() if (workspace is not None and need) else None
    ws_len = workspace.numel() * workspace.element_size() if (workspace is not None and need) else 0
    dm = desc(mask, F16) if mask is not None else None
    s = stream if stream is not None else torch.cuda.current_stream(q.device)
    rc = L.vtx_flash_attn_ext(ctypes.byref(dq), ctypes.byref(dk), ctypes.byref(dv),
                              ctypes.byref(dm) if dm is not None else None, ctypes.byref(p),
                              ctypes.byref(desc(out)), ws_ptr, ws_len, ctypes.c_void_p(s.cuda_stream))
    _check(rc, "vtx_flash_attn_ext")
    return out


class DecodeBatchPlan:
    """Device-side arrays for vtx_flash_attn_decode_batched over a fixed set of
    per-stream KV buffers (pointer arrays live on the device so one call can be
    captured in a CUDA graph and replayed)."""

    def __init__(self, k_bufs: Sequence[torch.Tensor], v_bufs: Sequence[torch.Tensor],
                 kv_len: torch.Tensor, n_head_q: int, n_head_kv: int, head_dim: int, kv_type: int,
                 kv_nb1: int, kv_nb2: int, max_kv_len: int, scale: float,
                 fresh_row: Optional[torch.Tensor] = None):
        """fresh_row: optional device int32 [n_seq], the row of each stream that
        the kernel launched just before each call writes (vtx_decode_batch)."""
        dev = kv_len.device
        self.k_ptrs = torch.tensor([t.data_ptr() for t in k_bufs], dtype=torch.int64, device=dev)
        self.v_ptrs = torch.tensor([t.data_ptr() for t in v_bufs], dtype=torch.int64, device=dev)
        self.kv_len = kv_len.to(torch.int32)
        self.keep = (list(k_bufs), list(v_bufs))
        b = DecodeBatch()
        b.n_seq, b.n_head_q, b.n_head_kv, b.head_dim = len(k_bufs), n_head_q, n_head_kv, head_dim
        b.kv_type, b.max_kv_len, b.kv_nb1, b.kv_nb2 = kv_type, max_kv_len, kv_nb1, kv_nb2
        b.k_ptrs, b.v_ptrs, b.kv_len = self.k_ptrs.data_ptr(), self.v_ptrs.data_ptr(), self.kv_len.data_ptr()
        b.scale = scale
        self.fresh_row = fresh_row
        b.fresh_row = fresh_row.data_ptr() if fresh_row is not None else None
        self.batch = b
        need = load().vtx_flash_attn_decode_batched_workspace(ctypes.byref(b))
        if need == ctypes.c_size_t(-1).value:
            raise VtxError(-3, "batch rejected")
        self.workspace = torch.empty(max(int(need), 1), dtype=torch.uint8, device=dev)
        self.need = int(need)

    def __call__(self, q: torch.Tensor, out: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        if out is None:
            out = _empty(q.shape, torch.float32, q.device, stream)
        self.batch.q = q.data_ptr()
        self.batch.dst = out.data_ptr()
        s = stream if stream is not None else torch.cuda.current_stream(q.device)
        rc = load().vtx_flash_attn_decode_batched(ctypes.byref(self.batch), self.workspace.data_ptr(),
                                                  self.workspace.numel(), ctypes.c_void_p(s.cuda_stream))
        _check(rc, "vtx_flash_attn_decode_batched")
        return out


def kv_append(k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
              k_cache: torch.Tensor, v_cache: torch.Tensor, kv_type: int, freq_base: float = 1e6, *,
              q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
              k_cache_ptrs: Optional[torch.Tensor] = None, v_cache_ptrs: Optional[torch.Tensor] = None,
              cache_nb1: Optional[int] = None, stream: Optional[torch.cuda.Stream] = None) -> Optional[torch.Tensor]:
    """vtx_kv_append: RoPE (ggml mode 0) of q and k, then k/v written into the
    cache rows ``slots`` (F32, F16 or Q8_0 bytes).  k, v: (T, Hkv, D) float32
    (heads contiguous), q: (T, Hq, D) float32 or None.  Caches: rows of
    Hkv * head bytes, ``cache_nb1`` bytes apart (default: the row size).
    Returns q_out (allocated when q is given and q_out is None)."""
    T, Hkv, D = k.shape
    for t in (k, v) + ((q,) if q is not None else ()):
        if t.dtype != torch.float32 or t.stride(2) != 1 or t.stride(1) != D:
            raise VtxError(-4, "q/k/v must be float32 with heads contiguous")
    if q is not None and q_out is None:
        q_out = _empty(q.shape, q.dtype, q.device, stream)
    a = KvAppendArgs()
    a.n_tokens, a.n_head_kv, a.head_dim, a.kv_type, a.freq_base = T, Hkv, D, kv_type, freq_base
    if q is not None:
        a.n_head_q, a.q, a.q_nb1 = q.shape[1], q.data_ptr(), q.stride(0) * 4
        a.q_out, a.q_out_nb1 = q_out.data_ptr(), q_out.stride(0) * 4
    a.k, a.k_nb1, a.v, a.v_nb1 = k.data_ptr(), k.stride(0) * 4, v.data_ptr(), v.stride(0) * 4
    with torch.cuda.stream(stream):                # copies, if any, are made and freed where they are read
        pos = positions.to(torch.int32).contiguous()
        sl = slots.to(torch.int32).contiguous()
    a.positions, a.slots = pos.data_ptr(), sl.data_ptr()
    a.k_cache = k_cache.data_ptr() if k_cache is not None else None
    a.v_cache = v_cache.data_ptr() if v_cache is not None else None
    a.k_cache_ptrs = k_cache_ptrs.data_ptr() if k_cache_ptrs is not None else None
    a.v_cache_ptrs = v_cache_ptrs.data_ptr() if v_cache_ptrs is not None else None
    if cache_nb1 is None:
        cache_nb1 = k_cache.stride(0) * k_cache.element_size()
    a.cache_nb1 = cache_nb1
    s = stream if stream is not None else torch.cuda.current_stream(k.device)
    _check(load().vtx_kv_append(ctypes.byref(a), ctypes.c_void_p(s.cuda_stream)), "vtx_kv_append")
    return q_out


class DecodeLayerPlan:
    """vtx_decode_layer over a fixed set of per-stream caches: RoPE of Q and K,
    the new K/V row into ring slot ``slots[s]`` and decode attention over rows
    [0, kv_len[s]), one launch per call.  The counters (positions, slots,
    kv_len) and the cache pointer arrays live on the device, so a call can be
    captured in a CUDA graph and replayed while the counters advance."""

    def __init__(self, k_bufs: Sequence[torch.Tensor], v_bufs: Sequence[torch.Tensor], positions: torch.Tensor,
                 slots: torch.Tensor, kv_len: torch.Tensor, n_head_q: int, n_head_kv: int, head_dim: int,
                 kv_type: int, cache_nb1: int, max_kv_len: int, scale: float, freq_base: float = 1e6,
                 early: bool = False):
        dev = kv_len.device
        self.k_ptrs = torch.tensor([t.data_ptr() for t in k_bufs], dtype=torch.int64, device=dev)
        self.v_ptrs = torch.tensor([t.data_ptr() for t in v_bufs], dtype=torch.int64, device=dev)
        self.keep = (list(k_bufs), list(v_bufs), positions, slots, kv_len)
        a = DecodeLayerArgs()
        a.n_seq, a.n_head_q, a.n_head_kv, a.head_dim = len(k_bufs), n_head_q, n_head_kv, head_dim
        a.kv_type, a.max_kv_len, a.freq_base, a.scale = kv_type, max_kv_len, freq_base, scale
        a.positions, a.slots, a.kv_len = positions.data_ptr(), slots.data_ptr(), kv_len.data_ptr()
        a.k_cache_ptrs, a.v_cache_ptrs, a.cache_nb1 = self.k_ptrs.data_ptr(), self.v_ptrs.data_ptr(), cache_nb1
        a.early = 1 if early else 0
        self.args = a
        need = load().vtx_decode_layer_workspace(ctypes.byref(a))
        if need == ctypes.c_size_t(-1).value:
            raise VtxError(-3, "decode layer rejected")
        self.need = int(need)
        # zeroed once: the split-arrival counters start at 0 and every call leaves them there
        self.workspace = torch.zeros(max(self.need, 1), dtype=torch.uint8, device=dev)

    def __call__(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """q: (n_seq, Hq, D), k/v: (n_seq, Hkv, D) float32, heads contiguous;
        returns (n_seq, Hq, D) float32."""
        for t in (q, k, v):
            if t.dtype != torch.float32 or t.stride(2) != 1 or t.stride(1) != t.shape[2]:
                raise VtxError(-4, "q/k/v must be float32 with heads contiguous")
        if out is None:
            out = _empty(q.shape, q.dtype, q.device, stream)
        a = self.args
        a.q, a.q_nb1 = q.data_ptr(), q.stride(0) * 4
        a.k, a.k_nb1 = k.data_ptr(), k.stride(0) * 4
        a.v, a.v_nb1 = v.data_ptr(), v.stride(0) * 4
        a.dst, a.dst_nb1 = out.data_ptr(), out.stride(0) * 4
        s = stream if stream is not None else torch.cuda.current_stream(q.device)
        _check(load().vtx_decode_layer(ctypes.byref(a), self.workspace.data_ptr(), self.workspace.numel(),
                                       ctypes.c_void_p(s.cuda_stream)), "vtx_decode_layer")
        return out


# ---- paged decoder cache ------------------------------------------------------

_ROW_TYPES = {torch.float32: (F32, 4), torch.float16: (F16, 2)}      # dtype -> (type id, bytes)


class PagedKv:
    """A decoder cache in pages with one step's ragged batch of new tokens
    (vtx_paged_kv), and the calls over it: append, attend, score, evict.

    k_pool, v_pool: (n_pages, n_head_kv, page_size, D) float16 views, or uint8
    with Q8_0 blocks on the last axis (rows of a head contiguous).  page_table:
    int32 (n_seq, max_pages), kv_len: int32 (n_seq,), q_start: int32
    (n_seq + 1,), contiguous on the pools' device: the kernels read them, so
    they may change between calls (and between replays of a captured call)
    within n_tokens, max_new and max_kv_len (default: the table's capacity; the
    tighter it is, the better the work is cut).  Workspaces are made here once
    (with a synchronisation, so outside of captures), up to 4 GiB where chunks
    meet a Q8_0 cache; share= takes those of another PagedKv, no smaller ones, so
    that layers, or prompts and single tokens, have one set between them.  Calls
    on one PagedKv, or on those that share, may come from several host threads,
    but must not overlap on the GPU, and it must live until they are done.  Inputs
    and outputs stay the caller's and are not copied.  A call with stream= is
    queued there and waits for nothing else: its inputs have to be ready on that
    stream, and a result that it makes is that stream's."""

    def __init__(self, k_pool: torch.Tensor, v_pool: torch.Tensor, page_table: torch.Tensor, kv_len: torch.Tensor,
                 q_start: torch.Tensor, n_head_q: int, *, n_tokens: int, max_new: int,
                 max_kv_len: Optional[int] = None, share: Optional["PagedKv"] = None):
        if k_pool.dim() != 4 or v_pool.shape != k_pool.shape or v_pool.dtype != k_pool.dtype or \
                v_pool.device != k_pool.device:
            raise VtxError(-3, "k_pool and v_pool must be (n_pages, n_head_kv, page_size, D) alike")
        if k_pool.dtype not in (torch.float16, torch.uint8):
            raise VtxError(-2, "pools must be float16 or Q8_0 bytes")
        self.dev, self._on = k_pool.device, k_pool.get_device()
        self._only = self.dev.type == "cuda" and torch.cuda.device_count() == 1      # always the current one
        n_seq = kv_len.shape[0]
        for t, shape in ((page_table, (n_seq, page_table.shape[-1])), (kv_len, (n_seq,)), (q_start, (n_seq + 1,))):
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != self.dev or tuple(t.shape) != shape:
                raise VtxError(-3, "page_table, kv_len and q_start must be contiguous int32 on the pools' device")
        self.k_pool, self.v_pool, self.page_table, self.kv_len, self.q_start = k_pool, v_pool, page_table, kv_len, q_start
        self.n_seq, self.n_head_q, self.n_head_kv = n_seq, n_head_q, k_pool.shape[1]
        kvt = Q8_0 if k_pool.dtype == torch.uint8 else F16
        self.head_dim = k_pool.shape[3] // Q8_0_BLOCK * QK8_0 if kvt == Q8_0 else k_pool.shape[3]
        self.n_tokens = n_tokens
        c = VtxPagedKv()
        c.k, c.v = self._pool(k_pool, kvt), self._pool(v_pool, kvt)
        c.page_table, c.kv_len, c.q_start = page_table.data_ptr(), kv_len.data_ptr(), q_start.data_ptr()
        c.n_seq, c.max_pages, c.n_tokens, c.max_new = n_seq, page_table.shape[1], n_tokens, max_new
        c.max_kv_len = page_table.shape[1] * k_pool.shape[2] if max_kv_len is None else max_kv_len
        self.c = c
        self.max_kv_len = c.max_kv_len
        self._lib = load()
        with torch.cuda.device(self.dev if self.dev.type == "cuda" else -1):     # plans follow the device's SMs
            need = [self._lib.vtx_flash_attn_paged_workspace(ctypes.byref(c), n_head_q),
                    self._lib.vtx_kv_evict_paged_workspace(ctypes.byref(c))]
        if ctypes.c_size_t(-1).value in need:
            raise VtxError(-3, "paged cache rejected")
        if share is not None:
            pairs = (n_seq * self.n_head_kv, share.n_seq * share.n_head_kv)
            if share.dev != self.dev or share.workspace.numel() < need[0] or share.evict_workspace.numel() < need[1] or \
                    (max(pairs) > 65536 and pairs[0] != pairs[1]):              # counters beyond their fixed place
                raise VtxError(-6, "the shared workspaces are too small, or on another device")
            self.workspace, self.evict_workspace = share.workspace, share.evict_workspace
        else:
            # attention's holds arrival counters: zero once, left zeroed by every call
            self.workspace = torch.zeros(max(need[0], 256), dtype=torch.uint8, device=self.dev)
            self.evict_workspace = torch.empty(max(need[1], 256), dtype=torch.uint8, device=self.dev)
            if self.dev.type == "cuda":             # the first call may be on another stream
                torch.cuda.current_stream(self.dev).synchronize()
        self._ws, self._evict_ws = ((w.data_ptr(), w.numel()) for w in (self.workspace, self.evict_workspace))
        # argument blocks, made once: a call only sets its tensors
        self._q_shape = (n_tokens, n_head_q, self.head_dim)
        self._kv_shape = (n_tokens, self.n_head_kv, self.head_dim)
        self._ones = 1 in (n_tokens, n_head_q, self.n_head_kv)
        self._q, self._dst, self._params = VtxTensor(), VtxTensor(), FaParams()
        for d in (self._q, self._dst):
            d.ne[0], d.ne[3] = self.head_dim, 1
        self._q.ne[1], self._q.ne[2] = n_tokens, n_head_q
        self._dst.ne[1], self._dst.ne[2] = n_head_q, n_tokens
        self._q_nb, self._dst_nb = self._q.nb, self._dst.nb
        at, adr = ctypes.addressof, ctypes.addressof(c)
        self._append, self._attend = KvAppendPagedArgs(), FlashAttnPagedArgs()
        self._score, self._evict = KvScorePagedArgs(), KvEvictPagedArgs()
        for a in (self._append, self._attend, self._score, self._evict):
            a.kv = adr
        self._lock = threading.Lock()               # a call fills its block and reads it, another thread's waits
        self._refs = [ctypes.byref(a) for a in (self._append, self._attend, self._score, self._evict)]
        self._attend.q, self._attend.dst, self._attend.params = at(self._q), at(self._dst), at(self._params)
        self._score.q, self._score.params = at(self._q), at(self._params)

    @staticmethod
    def _pool(t: torch.Tensor, kvt: int) -> VtxTensor:
        d = VtxTensor()
        es, s = t.element_size(), t.stride()
        if s[3] != 1:
            raise VtxError(-4, "the last axis of a pool must be contiguous")
        d.type = kvt
        row = t.shape[3] * es
        # an axis of one element: any legal stride
        nb = [34 if kvt == Q8_0 else es, s[2] * es, s[1] * es if t.shape[1] > 1 else row * t.shape[2], s[0] * es]
        if t.shape[0] == 1:
            nb[3] = max(nb[1] * t.shape[2], nb[2] * t.shape[1])
        ne = [t.shape[3] // Q8_0_BLOCK * QK8_0 if kvt == Q8_0 else t.shape[3], t.shape[2], t.shape[1], t.shape[0]]
        for i in range(4):
            d.ne[i], d.nb[i] = ne[i], nb[i]
        d.data = t.data_ptr()
        return d

    def _strides(self, t: torch.Tensor):
        """Strides, those of axes with one element (which may be anything) as if contiguous."""
        st = t.stride()
        if not self._ones or len(st) != 3:
            return st
        head = st[1] if t.shape[1] > 1 else t.shape[2]
        return st[0] if t.shape[0] > 1 else head * t.shape[1], head, st[2]

    def _rows(self, t: torch.Tensor, what: str, d: VtxTensor, nb, token: int, head: int) -> None:
        """Puts a (n_tokens, n_head_q, D) float32 / float16 view into descriptor d."""
        st, kind = self._strides(t), _ROW_TYPES.get(t.dtype)
        if t.shape != self._q_shape or st[2] != 1 or t.get_device() != self._on:
            raise VtxError(-3, f"{what} must be {self._q_shape} on {self.dev}, last axis contiguous")
        if kind is None:
            raise VtxError(-2, f"{what}: dtype {t.dtype}")
        d.type, es = kind
        nb[0], nb[token], nb[head], d.data = es, st[0] * es, st[1] * es, t.data_ptr()

    def _array(self, t: Optional[torch.Tensor], dtype: torch.dtype, what: str, cap: Optional[int]) -> Optional[int]:
        """Checks a (n_seq, n_head_kv, cap) row array; returns its cap."""
        if t is None:
            return cap
        shape = t.shape
        if len(shape) != 3 or shape[0] != self.n_seq or shape[1] != self.n_head_kv or t.dtype != dtype or \
                not t.is_contiguous() or t.get_device() != self._on or (cap is not None and shape[2] != cap):
            raise VtxError(-3, f"{what} must be a contiguous ({self.n_seq}, {self.n_head_kv}, rows) {dtype} tensor")
        return shape[2]

    def _set_params(self, scale, causal, window, softcap) -> None:
        p = self._params
        p.scale = self.head_dim ** -0.5 if scale is None else scale
        p.logit_softcap, p.causal, p.window = softcap, 1 if causal else 0, window

    def _call(self, fn, args, stream: Optional[torch.cuda.Stream], *ws) -> None:
        dev = self.dev
        if dev.type != "cuda":
            raise VtxError(-8, "the pools are not on a GPU")
        s = stream.cuda_stream if stream is not None else torch._C._cuda_getCurrentRawStream(self._on)
        if self._only or torch._C._cuda_getDevice() == self._on:
            rc = fn(args, *ws, s)
        else:
            with torch.cuda.device(dev):
                rc = fn(args, *ws, s)
        if rc != 0:
            raise VtxError(rc, fn.__name__)

    def append(self, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, freq_base: float = 1e6, *,
               q: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None,
               row_pos: Optional[torch.Tensor] = None, score: Optional[torch.Tensor] = None,
               stream: Optional[torch.cuda.Stream] = None) -> Optional[torch.Tensor]:
        """vtx_kv_append_paged: k, v (n_tokens, n_head_kv, D) float32 into the new
        tokens' rows, K rotated to positions (int32 (n_tokens,)); q (n_tokens,
        n_head_q, D) float32 rotated into q_out (float32 or float16; made as
        float16 when not given).  row_pos (int32) and score (float32),
        (n_seq, n_head_kv, rows): the new rows' entries are set."""
        D, a = self.head_dim, self._append
        ks, vs = self._strides(k), self._strides(v)
        if k.shape != self._kv_shape or v.shape != self._kv_shape or ks[2] != 1 or ks[1] != D or vs[2] != 1 or \
                vs[1] != D or k.dtype != torch.float32 or v.dtype != torch.float32:
            raise VtxError(-4, f"k and v must be {self._kv_shape} float32 with heads contiguous")
        if positions.dtype != torch.int32 or positions.shape != (self.n_tokens,) or not positions.is_contiguous():
            raise VtxError(-3, "positions must be contiguous int32, one per token")
        if not k.get_device() == v.get_device() == positions.get_device() == self._on:
            raise VtxError(-3, f"k, v and positions must be on {self.dev}")
        if q is not None:
            if q_out is None:
                q_out = _empty(q.shape, torch.float16, self.dev, stream)
            if not q.get_device() == q_out.get_device() == self._on:
                raise VtxError(-3, f"q and q_out must be on {self.dev}")
            qs, os_, kind = self._strides(q), self._strides(q_out), _ROW_TYPES.get(q_out.dtype)
            if q.shape != self._q_shape or q_out.shape != self._q_shape or qs[2] != 1 or qs[1] != D or os_[2] != 1 or \
                    os_[1] != D or q.dtype != torch.float32 or kind is None:
                raise VtxError(-4, f"q (float32) and q_out must be {self._q_shape} with heads contiguous")
        elif q_out is not None:
            raise VtxError(-1, "q_out without q")
        cap = self._array(score, torch.float32, "score", self._array(row_pos, torch.int32, "row_pos", None)) or 0
        with self._lock:
            if q is not None:
                a.n_head_q, (a.q_out_type, es) = self.n_head_q, kind
                a.q, a.q_nb1, a.q_out, a.q_out_nb1 = q.data_ptr(), qs[0] * 4, q_out.data_ptr(), os_[0] * es
            else:
                a.q = a.q_out = None
            a.freq_base, a.row_cap = freq_base, cap
            a.k, a.k_nb1, a.v, a.v_nb1 = k.data_ptr(), ks[0] * 4, v.data_ptr(), vs[0] * 4
            a.positions = positions.data_ptr()
            a.row_pos = row_pos.data_ptr() if row_pos is not None else None
            a.score = score.data_ptr() if score is not None else None
            self._call(self._lib.vtx_kv_append_paged, self._refs[0], stream)
        return q_out

    def attend(self, q: torch.Tensor, out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None, *,
               scale: Optional[float] = None, causal: bool = True, window: int = 0, logit_softcap: float = 0.0,
               stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """vtx_flash_attn_paged: q (n_tokens, n_head_q, D) float16 / float32 ->
        out, same shape (float32, or the type of the given tensor).  lse:
        optional float32 (n_tokens, n_head_q) that receives ln sum exp.  scale
        defaults to D ** -0.5.  Rows of tokens of no stream are left as they are
        (not initialised, in a result made here)."""
        if out is None:
            out = _empty(self._q_shape, torch.float32, self.dev, stream)
        with self._lock:
            self._rows(q, "q", self._q, self._q_nb, 1, 2)
            self._rows(out, "out", self._dst, self._dst_nb, 2, 1)
            self._set_params(scale, causal, window, logit_softcap)
            self._attend.lse = self._check_lse(lse) if lse is not None else None
            self._call(self._lib.vtx_flash_attn_paged, self._refs[1], stream, *self._ws)
        return out

    def _check_lse(self, lse: torch.Tensor) -> int:
        if lse.shape != self._q_shape[:2] or lse.dtype != torch.float32 or not lse.is_contiguous() or \
                lse.get_device() != self._on:
            raise VtxError(-3, f"lse must be a contiguous float32 (n_tokens, n_head_q) tensor on {self.dev}")
        return lse.data_ptr()

    def score(self, q: torch.Tensor, lse: torch.Tensor, score: torch.Tensor, score_out: Optional[torch.Tensor] = None,
              *, scale: Optional[float] = None, causal: bool = True, window: int = 0, logit_softcap: float = 0.0,
              observe: int = 0, decay: float = 1.0, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """vtx_kv_score_paged: adds the attention weight that the new tokens (the
        last ``observe`` of each stream; 0: all) gave every cached row to
        decay * score, float32 (n_seq, n_head_kv, rows); in place, or into
        score_out.  q and lse as attend read and wrote them."""
        out = score if score_out is None else score_out
        cap = self._array(out, torch.float32, "score_out", self._array(score, torch.float32, "score", None))
        a = self._score
        with self._lock:
            self._rows(q, "q", self._q, self._q_nb, 1, 2)
            self._set_params(scale, causal, window, logit_softcap)
            a.lse, a.score, a.score_out = self._check_lse(lse), score.data_ptr(), out.data_ptr()
            a.row_cap, a.observe, a.decay = cap, observe, decay
            self._call(self._lib.vtx_kv_score_paged, self._refs[2], stream)
        return out

    def evict(self, score: torch.Tensor, keep: int, kv_len_out: Optional[torch.Tensor] = None, *, n_sink: int = 0,
              n_recent: int = 0, row_pos: Optional[torch.Tensor] = None, next_pos: Optional[torch.Tensor] = None,
              score_out: Optional[torch.Tensor] = None, pos_out: Optional[torch.Tensor] = None,
              src_out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """vtx_kv_evict_paged: every (stream, KV head) keeps its ``keep`` best rows,
        moved together in place; kv_len_out (default: kv_len itself) receives
        the new lengths.  Where several caches (layers) share one kv_len, give
        each call another kv_len_out and copy it to kv_len after the last one:
        a shorter kv_len cuts off what the next cache still had to choose from.
        score_out, pos_out, src_out: optional
        (n_seq, n_head_kv, >= keep) arrays of the kept rows' scores, positions
        and old row indices; score_out may be score and pos_out row_pos."""
        if kv_len_out is None:
            kv_len_out = self.kv_len
        for t, what in ((kv_len_out, "kv_len_out"), (next_pos, "next_pos")):
            if t is not None and (t.dtype != torch.int32 or t.shape != (self.n_seq,) or not t.is_contiguous() or
                                  t.get_device() != self._on):
                raise VtxError(-3, f"{what} must be contiguous int32 on {self.dev}, one per stream")
        a = self._evict
        rows = self._array(row_pos, torch.int32, "row_pos", self._array(score, torch.float32, "score", None))
        cap = self._array(pos_out, torch.int32, "pos_out", self._array(score_out, torch.float32, "score_out", None))
        cap = self._array(src_out, torch.int32, "src_out", cap) or 0
        ptr = lambda t: t.data_ptr() if t is not None else None  # noqa: E731
        with self._lock:
            a.score, a.row_pos, a.next_pos, a.kv_len_out = score.data_ptr(), ptr(row_pos), ptr(next_pos), kv_len_out.data_ptr()
            a.score_out, a.pos_out, a.src_out = ptr(score_out), ptr(pos_out), ptr(src_out)
            a.keep, a.n_sink, a.n_recent, a.row_cap, a.out_cap = keep, n_sink, n_recent, rows, cap
            self._call(self._lib.vtx_kv_evict_paged, self._refs[3], stream, *self._evict_ws)
        return kv_len_out


# ---- realtime encoder: chunk plan and device-side stitch ---------------------

def encoder_chunk_plan(total_mel_frames: int):
    """The chunks run_encoder_chunked processes for an utterance
    (src/voxtral.cpp:2234-2335), through vtx_encoder_chunk_plan.  Returns
    (chunks as a ctypes array of EncChunk, stitched token count, count
    trimmed to a multiple of 4)."""
    L = load()
    tot, used = ctypes.c_int32(0), ctypes.c_int32(0)
    n = L.vtx_encoder_chunk_plan(int(total_mel_frames), None, 0, ctypes.byref(tot), ctypes.byref(used))
    _check(n if n < 0 else 0, "vtx_encoder_chunk_plan")
    arr = (EncChunk * max(n, 1))()
    n2 = L.vtx_encoder_chunk_plan(int(total_mel_frames), arr, n, ctypes.byref(tot), ctypes.byref(used))
    _check(n2 if n2 < 0 else 0, "vtx_encoder_chunk_plan")
    return (EncChunk * n).from_buffer(arr) if n else (EncChunk * 0)(), tot.value, used.value


def encoder_stitch(chunk_out: torch.Tensor, chunks, dst: torch.Tensor,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Copies rows [skip, skip + stride) of each chunk's output into rows
    [write_offset, ...) of dst on the device (vtx_encoder_stitch).
    chunk_out: (n_chunks, rows, ...) with contiguous rows; dst: (rows_total, ...)."""
    if chunk_out.shape[0] < len(chunks):
        raise ValueError("fewer chunk outputs than chunks")
    row_bytes = chunk_out[0, 0].numel() * chunk_out.element_size()
    if dst[0].numel() * dst.element_size() != row_bytes or not chunk_out[0, 0].is_contiguous():
        raise ValueError("row size mismatch or non-contiguous rows")
    s = stream if stream is not None else torch.cuda.current_stream()
    arr = (EncChunk * max(len(chunks), 1))(*chunks) if len(chunks) else (EncChunk * 1)()
    rc = load().vtx_encoder_stitch(ctypes.c_void_p(chunk_out.data_ptr()), chunk_out.stride(0) * chunk_out.element_size(),
                                   chunk_out.stride(1) * chunk_out.element_size(), ctypes.c_void_p(dst.data_ptr()),
                                   dst.stride(0) * dst.element_size(), row_bytes, arr, len(chunks),
                                   ctypes.c_void_p(s.cuda_stream))
    _check(rc, "vtx_encoder_stitch")
    return dst


def read_device_error(stream: Optional[torch.cuda.Stream] = None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return int(load().vtx_read_device_error(ctypes.c_void_p(s.cuda_stream)))


# ---- reference masks and formats (the shapes voxtral.cpp builds) -----------

def causal_mask(n: int, device=None) -> torch.Tensor:
    """src/voxtral.cpp:2103-2111 fill_causal_mask -> F16 (:1801)."""
    m = torch.full((n, n), float("-inf"), device=device).triu(1)
    return m.to(torch.float16)


def window_mask(n: int, window: int = 750, device=None) -> torch.Tensor:
    """src/voxtral.cpp:2181-2188 chunk-local sliding causal mask -> F16."""
    qi = torch.arange(n, device=device)[:, None]
    kj = torch.arange(n, device=device)[None, :]
    allow = (kj <= qi) & (kj >= (qi - (window - 1)).clamp(min=0))
    return torch.where(allow, 0.0, float("-inf")).to(torch.float16)


def quantize_q8_0(x: torch.Tensor) -> torch.Tensor:
    """ggml's reference Q8_0 quantizer (quantize_row_q8_0_ref, the rule the
    reference's converter uses for Q8_0 tensors) over the last axis of a float
    tensor, on x's device: per 32 values d = amax/127 (stored as f16),
    q = round-half-away(x / d).  Returns uint8 with the last axis holding
    D/32 blocks of 34 bytes {f16 d; int8 qs[32]}.  A data-preparation helper
    for caches built outside vtx_kv_append (which quantizes on write)."""
    D = x.shape[-1]
    if D % QK8_0:
        raise VtxError(-3, "last axis must be a multiple of 32")
    xb = x.float().reshape(*x.shape[:-1], D // QK8_0, QK8_0)
    d = xb.abs().amax(dim=-1) / 127.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    y = xb * inv.unsqueeze(-1)
    qs = (torch.sign(y) * torch.floor(y.abs() + 0.5)).to(torch.int8)
    out = torch.empty(*x.shape[:-1], D // QK8_0, Q8_0_BLOCK, dtype=torch.uint8, device=x.device)
    out[..., :2] = d.half().unsqueeze(-1).view(torch.uint8).reshape(*d.shape, 2)
    out[..., 2:] = qs.view(torch.uint8)
    return out.reshape(*x.shape[:-1], D // QK8_0 * Q8_0_BLOCK)


def _raw_tensor(ttype: int, ne, nb, ptr: int) -> VtxTensor:
    d = VtxTensor()
    d.type = ttype
    for i in range(4):
        d.ne[i] = ne[i] if i < len(ne) else 1
        d.nb[i] = nb[i] if i < len(nb) else (d.nb[i - 1] * d.ne[i - 1])
    d.data = ptr
    return d


def out_proj(attn: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor] = None,
             residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
             stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """vtx_attn_out_proj: out = residual + bias + f16(attn) @ w^T (f32 accumulate),
    the output projection after the attention node (src/voxtral.cpp:1612-1617,
    :1804-1809).  attn: (1, n, Hq, Dv) float32 as flash_attn_ext returns it,
    any strides, read in place, or float16 (flash_attn_ext with a float16
    `out`: the same rounding, done in the attention epilogue); or
    (1, n, R, h, Dv), the rank-major result of shard.head_split_prefill
    (head = r * h + j).  w: (N, Hq * Dv) float16;
    bias: (N,) float32 or None; residual: (n, N) float32 or None (it may be
    `out`).  Returns out (n, N) float32."""
    if attn.dtype not in (torch.float32, torch.float16) or w.dtype != torch.float16:
        raise VtxError(-2, "attn must be float32 or float16 and w float16")
    es = attn.element_size()
    if attn.dim() == 4:
        _, n, Hq, Dv = attn.shape
        head_nb, tok_nb = attn.stride(2) * es, attn.stride(1) * es
        head_block, block_nb = 0, 0
    elif attn.dim() == 5:
        _, n, R, h, Dv = attn.shape
        Hq = R * h
        head_nb, tok_nb = attn.stride(3) * es, attn.stride(1) * es
        head_block, block_nb = h, attn.stride(2) * es
    else:
        raise VtxError(-3, "attn must be (1, n, Hq, Dv) or (1, n, R, h, Dv)")
    if attn.shape[0] != 1 or attn.stride(-1) != 1:
        raise VtxError(-3, "one batch, unit-stride head dim")
    N, K = w.shape
    if out is None:
        out = _empty((n, N), torch.float32, attn.device, stream)
    a = _raw_tensor(F32 if es == 4 else F16, [Dv, Hq, n, 1], [es, head_nb, tok_nb, tok_nb * n], attn.data_ptr())
    wd = _raw_tensor(F16, [K, N, 1, 1], [2, w.stride(0) * 2], w.data_ptr())
    yd = _raw_tensor(F32, [N, n, 1, 1], [4, out.stride(0) * 4], out.data_ptr())
    bd = _raw_tensor(F32, [N, 1, 1, 1], [4], bias.data_ptr()) if bias is not None else None
    rd = _raw_tensor(F32, [N, n, 1, 1], [4, residual.stride(0) * 4], residual.data_ptr()) \
        if residual is not None else None
    args = OutProjArgs()
    args.attn = ctypes.addressof(a)
    args.head_block, args.block_nb = head_block, block_nb
    args.w = ctypes.addressof(wd)
    args.bias = ctypes.addressof(bd) if bd is not None else None
    args.residual = ctypes.addressof(rd) if rd is not None else None
    args.dst = ctypes.addressof(yd)
    s = stream if stream is not None else torch.cuda.current_stream(attn.device)
    _check(load().vtx_attn_out_proj(ctypes.byref(args), ctypes.c_void_p(s.cuda_stream)), "vtx_attn_out_proj")
    return out
