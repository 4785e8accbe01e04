"""ctypes binding of libie_amd.so (include/ie_amd.h) for tests and benchmarks.

The product is the C ABI; this module only marshals torch device tensors into
it.  It never falls back to anything: if the HIP library is missing or a call
is rejected, it raises.
"""
from __future__ import annotations

import ctypes
import numbers
import os
from typing import NamedTuple

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libie_amd.so")

IE_OK, IE_ERR_INVALID, IE_ERR_UNSUPPORTED, IE_ERR_WORKSPACE, IE_ERR_HIP = range(5)
EPI_PLAIN, EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_RESIDUAL, EPI_I32 = range(5)
PATH_AUTO, PATH_GEMV, PATH_MFMA = range(3)
KV_F32, KV_BF16 = 0, 1
KV_I8 = 2  # Engine's kv_dtype only (include/ie_kv8.h)
BACKEND_INT8, BACKEND_FP32 = 0, 1
DA_REF_MAX_SPLITS = 16
DA_MAX_SPLITS = 256

_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_Z = ctypes.c_size_t

# name -> (restype, argtypes); mirrors include/ie_amd.h one to one.
SIGNATURES = {
    "ie_last_error": (ctypes.c_char_p, []),
    "ie_version": (_I, []),
    "ie_init": (_I, []),
    "ie_quantize_fp32_to_int8": (_I, [_I, _I, _P, _P, _P, _P]),
    "ie_int8_gemm": (_I, [_I, _I, _I, _P, _P, _P, _P, _I, _P, _P, _P, _P]),
    "ie_int8_gemm_ex": (_I, [_I, _I, _I, _P, _P, _P, _P, _I, _P, _P, _P, _I, _P]),
    "ie_decode_num_splits": (_I, [_I, _I, _I]),
    "ie_decode_attn_workspace_bytes": (_Z, [_I, _I, _I, _I]),
    "ie_decode_attn": (_I, [_I, _I, _I, _I, _P, _P, _P, _I, _P, _P, _I, _I, _I, _P, _P, _Z, _I, _P]),
    "ie_prefill_attn": (_I, [_I, _I, _I, _I, _I, _P, _P, _P, _I, _P, _I, _I, _I, _P, _P]),
    "ie_flash_attn": (_I, [_I, _I, _I, _I, _P, _P, _P, _P, _I, _P]),
    "ie_kv_cache_write": (_I, [_P, _P, _P, _P, _I, _P, _I, _I, _I, _I, _I, _P]),
    "ie_kv_cache_append_batch": (_I, [_I, _P, _P, _P, _P, _I, _P, _I, _P, _I, _I, _I, _P]),
    "ie_layernorm": (_I, [_I, _I, _P, _P, _P, _P, _F, _P]),
    "ie_layernorm_residual": (_I, [_I, _I, _P, _P, _P, _P, _P, _P, _F, _P]),
    "ie_embedding": (_I, [_P, _I, _I, _I, _P, _P, _P, _P]),
    "ie_embedding_batch": (_I, [_I, _P, _P, _I, _P, _P, _P, _P]),
    "ie_vocab_proj": (_I, [_I, _P, _P, _P, _I, _I, _P]),
    "ie_argmax": (_I, [_I, _P, _I, _P, _P]),
    "ie_topk": (_I, [_I, _P, _I, _I, _P, _P, _P]),
    "ie_top_k_draw": (_I, [_P, _P, _I, _F, ctypes.c_uint, _P]),
    "ie_check_token_ids": (_I, [_I, _P, _I]),
    "ie_decode_attn_noalloc": (_I, [_I, _I, _I, _I, _P, _P, _P, _I, _P, _P, _I, _I, _I, _P, _I, _P]),
}
DECODE_SCRATCH_BYTES = 32 << 20

# include/ie_kv8.h
KV8_SIGNATURES = {
    "ie_kv8_cache_write": (_I, [_I, _I, _P, _P, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P]),
    "ie_kv8_cache_append_batch": (_I, [_I, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _I, _I, _I, _P]),
    "ie_kv8_cache_read": (_I, [_I, _I, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P, _P, _P]),
    "ie_decode_kv8_num_splits": (_I, [_I, _I, _I, _I, _I, _I]),
    "ie_decode_attn_kv8": (_I, [_I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _P, _Z, _I, _P]),
    "ie_prefill_kv8_workspace_bytes": (_Z, [_I, _I, _I, _I, _I, _I]),
    "ie_prefill_attn_kv8": (_I, [_I, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _P, _Z, _P]),
}
KV8_MAX_SPLITS = 64

# include/ie_logprobs.h
LOGPROBS_SIGNATURES = {
    "ie_token_logprobs_workspace_bytes": (_Z, [_I, _I, _I]),
    "ie_token_logprobs": (_I, [_I, _P, _I, _I, _P, _I, _P, _P, _P, _P, _P, _P, _Z, _P]),
    "ie_engine_score": (_I, [_P, _I, _I, _P, _I, _P, _P, _P, _P, _P]),
}
LOGPROBS_TOP_MAX = 128

# include/ie_engine.h
ENGINE_SIGNATURES = {
    "ie_engine_create": (_I, [ctypes.POINTER(_P), ctypes.c_char_p, _I, _I, _I, _I, _I, _I,
                              ctypes.c_ulonglong, _I, _I, _I, _I, _I, _I, _I, _I]),
    "ie_engine_destroy": (_I, [_P]),
    "ie_engine_write_random_model": (_I, [ctypes.c_char_p, _I, _I, _I, _I, _I, _I, ctypes.c_ulonglong]),
    "ie_engine_reset": (_I, [_P]),
    "ie_engine_generate": (_I, [_P, _I, _I, _P, _I, _I, _P, _P]),
    "ie_engine_generate_one": (_I, [_P, _I, _P, _I, _F, _I, _I, _I, _P, _P, _P]),
    "ie_engine_step": (_I, [_P, _I, _P, _P, _P]),
    "ie_engine_prefill": (_I, [_P, _I, _I, _P, _P, _P]),
    "ie_engine_session_tokens": (_I, [_P]),
    "ie_engine_config": (_I, [_P, _P]),
    "ie_engine_step_bytes": (ctypes.c_double, [_P, _I]),
}


# include/ie_tokenizer.h (host code; no GPU)
TOKENIZER_SIGNATURES = {
    "ie_tokenizer_create": (_I, [_P, ctypes.c_char_p]),
    "ie_tokenizer_destroy": (_I, [_P]),
    "ie_tokenizer_encode": (_I, [_P, ctypes.c_char_p, _Z, _P, _Z, _P]),
    "ie_tokenizer_decode": (_I, [_P, _P, _Z, _P, _Z, _P]),
    "ie_tokenizer_vocab_size": (_I, [_P]),
    "ie_tokenizer_eos_token": (_I, [_P]),
}


class Metrics(ctypes.Structure):
    """ie_metrics (include/ie_engine.h): InferenceMetrics without `generating`."""
    _fields_ = [(n, ctypes.c_float) for n in ("ttft_ms", "tpot_ms", "itl_min_ms", "itl_max_ms",
                                              "itl_p95_ms", "tps")] + \
               [("tokens_generated", ctypes.c_int), ("max_tokens", ctypes.c_int)] + \
               [(n, ctypes.c_float) for n in ("kv_cache_pct", "vram_used_mb", "vram_total_mb", "mbu",
                                              "end_to_end_ms")]

    def as_dict(self):
        return {k: getattr(self, k) for k, _ in self._fields_}


class IeError(RuntimeError):
    def __init__(self, fn: str, status: int, msg: str):
        super().__init__(f"{fn} failed with status {status}: {msg}")
        self.status = status
        self.msg = msg


_lib = None
_fns: dict = {}  # entry points by name, filled by load()


def load() -> ctypes.CDLL:
    """Loads libie_amd.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        # torch ships its own libamdhip64 (file libamdhip64.so, soname
        # libamdhip64.so.7).  Loading torch first makes the dynamic loader bind
        # our libamdhip64.so.7 dependency to that copy; the other order maps
        # two HIP/HSA runtimes into the process and the second sees no device.
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} is missing: build it with __graft_entry__.build() "
                "(make -C cuda-llm-inference-engine_amd)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in (list(SIGNATURES.items()) + list(ENGINE_SIGNATURES.items())
                                  + list(TOKENIZER_SIGNATURES.items()) + list(KV8_SIGNATURES.items())
                                  + list(LOGPROBS_SIGNATURES.items())):
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
            _fns[name] = fn
        _lib = lib
    return _lib


def last_error() -> str:
    return load().ie_last_error().decode()


def call(name: str, *args) -> int:
    """Calls an ie_* entry point and returns its status without raising."""
    fn = _fns.get(name)
    if fn is None:
        fn = getattr(load(), name)
    return fn(*args)


def check(name: str, *args) -> None:
    fn = _fns.get(name)
    st = fn(*args) if fn is not None else call(name, *args)
    if st != IE_OK:
        raise IeError(name, st, last_error())


# ---------------------------------------------------------------- torch glue
# A call's own cost matters here: a decode step's small operations take 2-5 us
# on the GPU.  Pointers and the stream cross as plain integers (the argument
# types convert them), the current stream is read without building a stream
# object, and torch is imported only where a wrapper allocates: 7.2 -> 3.9 us
# for a quantizer call, of which the launch itself is about 3.
def _ptr(t):
    return None if t is None else t.data_ptr()


_raw_stream = None  # () -> handle of the current device's current stream


def _bind_raw_stream():
    global _raw_stream
    import torch

    torch.cuda.current_stream()  # initialises the device as a first use does
    get_device, get_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    _raw_stream = lambda: get_stream(get_device())  # noqa: E731
    return _raw_stream


def _stream(stream=None):
    if stream is not None:
        return stream.cuda_stream
    return (_raw_stream or _bind_raw_stream())()


def quantize(x, out_packed=None, out_scales=None, stream=None):
    """x: [rows, cols] fp32 cuda -> (packed int32 [rows, cols/4], scales [rows])."""
    rows, cols = x.shape
    if out_packed is None or out_scales is None:
        import torch

        if out_packed is None:
            out_packed = torch.empty((rows, cols // 4), dtype=torch.int32, device=x.device)
        if out_scales is None:
            out_scales = torch.empty(rows, dtype=torch.float32, device=x.device)
    check("ie_quantize_fp32_to_int8", rows, cols, x.data_ptr(), out_packed.data_ptr(), out_scales.data_ptr(),
          _stream(stream))
    return out_packed, out_scales


def int8_gemm(A_packed, BT_packed, sA=None, sB=None, epilogue=EPI_PLAIN, bias=None,
              residual=None, out=None, path=PATH_AUTO, stream=None):
    """Returns C [M, N] (fp32, or int32 for EPI_I32)."""
    M, K4 = A_packed.shape
    N = BT_packed.shape[0]
    if out is None:
        import torch

        dt = torch.int32 if epilogue == EPI_I32 else torch.float32
        out = torch.empty((M, N), dtype=dt, device=A_packed.device)
    check("ie_int8_gemm_ex", M, N, 4 * K4, _ptr(A_packed), _ptr(BT_packed), _ptr(sA), _ptr(sB),
          epilogue, _ptr(bias), _ptr(residual), _ptr(out), path, _stream(stream))
    return out


def num_splits(max_ctx: int, block_size: int, splits: int = 0) -> int:
    return call("ie_decode_num_splits", max_ctx, block_size, splits)


def workspace_bytes(B: int, H_q: int, d: int, splits: int) -> int:
    return call("ie_decode_attn_workspace_bytes", B, H_q, d, splits)


def decode_attn(Q, k_cache, v_cache, block_table, context_lens, max_ctx, block_size, H_kv,
                kv_dtype=KV_F32, splits=0, out=None, workspace=None, stream=None):
    """Q [B, H_q, d] fp32; caches [P, bs, H_kv, d]; returns O [B, H_q, d]."""
    B, H_q, d = Q.shape
    nbps = block_table.shape[1]
    if workspace is None:
        import torch

        need = workspace_bytes(B, H_q, d, num_splits(max_ctx, block_size, splits))
        workspace = torch.empty(max(need // 4, 1), dtype=torch.float32, device=Q.device)
    if out is None:
        import torch

        out = torch.empty_like(Q)
    check("ie_decode_attn", B, H_q, H_kv, d, _ptr(Q), _ptr(k_cache), _ptr(v_cache), kv_dtype,
          _ptr(block_table), _ptr(context_lens), max_ctx, block_size, nbps, _ptr(out),
          _ptr(workspace), workspace.numel() * 4, splits, _stream(stream))
    return out


def decode_attn_noalloc(Q, k_cache, v_cache, block_table, context_lens, max_ctx, block_size, H_kv,
                        kv_dtype=KV_F32, splits=0, out=None, stream=None):
    """ie_decode_attn_noalloc: as decode_attn, split partials in the library's
    per-device scratch (no workspace)."""
    B, H_q, d = Q.shape
    if out is None:
        import torch

        out = torch.empty_like(Q)
    check("ie_decode_attn_noalloc", B, H_q, H_kv, d, _ptr(Q), _ptr(k_cache), _ptr(v_cache), kv_dtype,
          _ptr(block_table), _ptr(context_lens), max_ctx, block_size, block_table.shape[1], _ptr(out),
          splits, _stream(stream))
    return out


def prefill_attn(Q, k_cache, v_cache, block_table, start_pos, block_size, H_kv, kv_dtype=KV_F32,
                 out=None, stream=None):
    """Q [B, P, H_q, d] fp32 (token t at position start_pos + t, its K/V already
    cached); returns causal O [B, P, H_q, d]."""
    B, P, H_q, d = Q.shape
    if out is None:
        import torch

        out = torch.empty_like(Q)
    check("ie_prefill_attn", B, P, H_q, H_kv, d, _ptr(Q), _ptr(k_cache), _ptr(v_cache), kv_dtype,
          _ptr(block_table), block_table.shape[1], block_size, start_pos, _ptr(out), _stream(stream))
    return out


def flash_attn(Q, K, V, causal=True, out=None, stream=None):
    """Q, K, V [B, H, N, d] fp32 -> O [B, H, N, d] (run_flash_attn_v2)."""
    B, H, N, d = Q.shape
    if out is None:
        import torch

        out = torch.empty_like(Q)
    check("ie_flash_attn", B, H, N, d, _ptr(Q), _ptr(K), _ptr(V), _ptr(out), int(causal), _stream(stream))
    return out


def kv_cache_write(K, V, k_cache, v_cache, block_table, start_pos, block_size,
                   kv_dtype=KV_F32, stream=None):
    seq, H, dh = K.shape
    check("ie_kv_cache_write", _ptr(K), _ptr(V), _ptr(k_cache), _ptr(v_cache), kv_dtype,
          _ptr(block_table), seq, start_pos, H, dh, block_size, _stream(stream))


def kv_cache_append_batch(K, V, k_cache, v_cache, block_table, positions, block_size,
                          kv_dtype=KV_F32, stream=None):
    B, H, dh = K.shape
    check("ie_kv_cache_append_batch", B, _ptr(K), _ptr(V), _ptr(k_cache), _ptr(v_cache), kv_dtype,
          _ptr(block_table), block_table.shape[1], _ptr(positions), H, dh, block_size,
          _stream(stream))


def layernorm(x, gamma, beta, out=None, eps=1e-5, stream=None):
    rows, cols = x.shape
    if out is None:
        import torch

        out = torch.empty_like(x)
    check("ie_layernorm", rows, cols, _ptr(x), _ptr(gamma), _ptr(beta), _ptr(out), eps, _stream(stream))
    return out


def layernorm_residual(x, residual, gamma, beta, out=None, residual_out=None, eps=1e-5, stream=None):
    """(LayerNorm(x + residual), x + residual); out / residual_out may alias
    the inputs."""
    rows, cols = x.shape
    if out is None or residual_out is None:
        import torch

        out = torch.empty_like(x) if out is None else out
        residual_out = torch.empty_like(x) if residual_out is None else residual_out
    check("ie_layernorm_residual", rows, cols, _ptr(x), _ptr(residual), _ptr(gamma), _ptr(beta), _ptr(out),
          _ptr(residual_out), eps, _stream(stream))
    return out, residual_out


def embedding(ids, start_pos, wte, wpe, out=None, stream=None):
    import torch

    seq = ids.shape[0]
    d = wte.shape[1]
    out = out if out is not None else torch.empty((seq, d), dtype=torch.float32, device=wte.device)
    check("ie_embedding", _ptr(ids), seq, start_pos, d, _ptr(wte), _ptr(wpe), _ptr(out), _stream(stream))
    return out


def vocab_proj(h, wte, out=None, stream=None):
    rows, d = h.shape
    V = wte.shape[0]
    if out is None:
        import torch

        out = torch.empty((rows, V), dtype=torch.float32, device=h.device)
    check("ie_vocab_proj", rows, _ptr(h), _ptr(wte), _ptr(out), d, V, _stream(stream))
    return out


def argmax(logits, out=None, stream=None):
    import torch

    rows, n = logits.shape
    out = out if out is not None else torch.empty(rows, dtype=torch.int32, device=logits.device)
    check("ie_argmax", rows, _ptr(logits), n, _ptr(out), _stream(stream))
    return out


def topk(logits, k, stream=None):
    """(values [rows, k] fp32, indices [rows, k] int32) of the k largest per row,
    by value descending, equal values by index ascending."""
    import torch

    rows, n = logits.shape
    vals = torch.empty((rows, k), dtype=torch.float32, device=logits.device)
    idx = torch.empty((rows, k), dtype=torch.int32, device=logits.device)
    check("ie_topk", rows, _ptr(logits), n, k, _ptr(vals), _ptr(idx), _stream(stream))
    return vals, idx


def top_k_draw(vals, idx, temperature, seed):
    """Host draw of sample_top_k over sorted (value, index) pairs (numpy)."""
    import numpy as np

    v = np.ascontiguousarray(vals, dtype=np.float32)
    i = np.ascontiguousarray(idx, dtype=np.int32)
    tok = ctypes.c_int(-1)
    check("ie_top_k_draw", v.ctypes.data, i.ctypes.data, len(v), ctypes.c_float(temperature),
          ctypes.c_uint(seed), ctypes.addressof(tok))
    return tok.value


# ------------------------------------------- 8-bit KV cache, log probabilities
def _refuse(what, *tensors):
    raise ValueError(f"{what}: needs contiguous tensors on cuda:{_device_index()} of the documented types and shapes, got "
                     + ", ".join(f"{t.dtype} {tuple(t.shape)} strides {tuple(t.stride())} on {t.device}" for t in tensors))


_device_index = None  # () -> index of the current device
_raw_stream_of = None  # device index -> handle of its current stream
_f32 = _i32 = _i8 = _empty = None


def _bind_torch():
    global _device_index, _raw_stream_of, _f32, _i32, _i8, _empty
    import torch

    load()  # fills _fns
    torch.cuda.current_stream()
    _f32, _i32, _i8, _empty = torch.float32, torch.int32, torch.int8, torch.empty
    _raw_stream_of = torch._C._cuda_getCurrentRawStream
    _device_index = torch._C._cuda_getDevice


def _failed(name, status):
    raise IeError(name, status, last_error())


def _past_int(what, name, value):  # (ctypes takes an int's lowest 32 bits and says nothing)
    raise ValueError(f"{what}: {name}={value} lies outside 32 bits")


def _new(stream, shape, dtype, device):
    """A tensor for a call on the given stream (None: the current one), of that
    stream's memory: what another stream still does with memory it gave back
    cannot meet it, nor can a later call there with this tensor's once freed."""
    if stream is None:
        return _empty(shape, dtype=dtype, device=device)
    import torch

    with torch.cuda.stream(stream):
        return _empty(shape, dtype=dtype, device=device)


class Kv8Cache(NamedTuple):
    """The paged KV cache in 8 bits (include/ie_kv8.h has the layout): K codes
    [pages, heads, block, d] and V codes [pages, heads, block / 16, d, 16] int8,
    scales [pages, heads] fp32."""
    k: "torch.Tensor"  # noqa: F821
    v: "torch.Tensor"  # noqa: F821
    k_scale: "torch.Tensor"  # noqa: F821
    v_scale: "torch.Tensor"  # noqa: F821

    @classmethod
    def empty(cls, pages, heads, d, block_size=16, device="cuda"):
        import torch

        return cls(torch.empty((pages, heads, block_size, d), dtype=torch.int8, device=device),
                   torch.empty((pages, heads, block_size // 16, d, 16), dtype=torch.int8, device=device),
                   torch.empty((pages, heads), dtype=torch.float32, device=device),
                   torch.empty((pages, heads), dtype=torch.float32, device=device))

    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in self)


# The wrappers' checks and calls are spelled out flat: an attribute of a tensor costs
# 50 to 85 ns, its shape, a helper call, a loop over tensors or a call by *args two to
# five times that, and a decode step's calls are about as long on the GPU as here.
# Contiguous tensors are compared by their numbers of elements.
def _kv8(what, cache, table):
    """(heads, block size, d, device, table's rows and columns) of a cache whose tensors fit each other."""
    if _device_index is None:
        _bind_torch()
    k, v, ks, vs = cache
    at = _device_index()
    pages, H, bs, d = k.shape
    if not (k.dtype is _i8 and v.dtype is _i8 and ks.dtype is _f32 and vs.dtype is _f32 and table.dtype is _i32
            and k.get_device() == at and v.get_device() == at and ks.get_device() == at and vs.get_device() == at
            and table.get_device() == at and k.is_contiguous() and v.is_contiguous() and ks.is_contiguous()
            and vs.is_contiguous() and table.is_contiguous() and v.numel() == pages * H * bs * d
            and ks.numel() == pages * H and vs.numel() == pages * H and table.dim() == 2):
        _refuse(what, k, v, ks, vs, table)
    rows, nbps = table.shape
    return H, bs, d, at, rows, nbps


def _kv8_rows(what, K, V, lead, H, d, at):
    """Distance between rows [*lead, H, d] fp32 that may lie apart (the columns
    of a QKV projection) but evenly so."""
    st = K.stride()
    if lead[-1] > 1:
        ld = st[len(lead) - 1]
    else:
        ld = st[0] if lead[0] > 1 else H * d
    want = (*lead, H, d)
    if (K.shape != want or V.shape != want or K.dtype is not _f32 or V.dtype is not _f32 or K.get_device() != at
            or V.get_device() != at or V.stride() != st or st[-1] != 1 or (H > 1 and st[-2] != d) or ld > 0x7FFFFFFF
            or (len(lead) == 2 and lead[0] > 1 and lead[1] > 1 and st[0] != lead[1] * ld)):
        raise ValueError(f"{what}: K and V need to be fp32 {want} on cuda:{at} with equal strides, rows whole and evenly "
                         f"spaced; got {tuple(K.shape)} strides {st}, {tuple(V.shape)} strides {V.stride()}")
    return ld


def kv8_cache_write(K, V, cache, block_table, start_pos, stream=None):
    """Rows K, V [B, P, heads, d] fp32 (views into a QKV projection serve as they
    lie) to positions start_pos .. of the sequences of block_table [B, nbps]."""
    H, bs, d, at, rows, nbps = _kv8("kv8_cache_write", cache, block_table)
    B, P = K.shape[:2]
    if rows != B:
        raise ValueError("kv8_cache_write: block_table has other sequences than K")
    if not -0x80000000 <= start_pos <= 0x7FFFFFFF:
        _past_int("kv8_cache_write", "start_pos", start_pos)
    ld = _kv8_rows("kv8_cache_write", K, V, (B, P), H, d, at) if B * P else H * d
    k, v, ks, vs = cache
    st = _fns["ie_kv8_cache_write"](
        B, P, K.data_ptr(), V.data_ptr(), ld, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(),
        block_table.data_ptr(), nbps, start_pos, H, d, bs, _raw_stream_of(at) if stream is None else stream.cuda_stream)
    if st:
        _failed("ie_kv8_cache_write", st)


def kv8_cache_append_batch(K, V, cache, block_table, positions, stream=None):
    """One row of each sequence, K, V [B, heads, d], to positions[b] (int32)."""
    H, bs, d, at, B, nbps = _kv8("kv8_cache_append_batch", cache, block_table)
    if (positions.numel() != B or positions.dtype is not _i32 or positions.get_device() != at
            or not positions.is_contiguous()):
        _refuse("kv8_cache_append_batch", K, block_table, positions)
    ld = _kv8_rows("kv8_cache_append_batch", K, V, (B,), H, d, at) if B else H * d
    k, v, ks, vs = cache
    st = _fns["ie_kv8_cache_append_batch"](
        B, K.data_ptr(), V.data_ptr(), ld, k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(),
        block_table.data_ptr(), nbps, positions.data_ptr(), H, d, bs,
        _raw_stream_of(at) if stream is None else stream.cuda_stream)
    if st:
        _failed("ie_kv8_cache_append_batch", st)


def kv8_cache_read(cache, block_table, starts, context_lens, n, out=None, stream=None):
    """(K, V) [B, n, heads, d] fp32: positions starts[b] .. starts[b] + n - 1 of each
    sequence, zeros from context_lens[b] on (None: no limit)."""
    H, bs, d, at, B, nbps = _kv8("kv8_cache_read", cache, block_table)
    if out is None:
        out = tuple(_new(stream, (B, n, H, d), _f32, cache[0].device) for _ in range(2))
    K, V = out
    size = B * n * H * d
    if not (starts.numel() == B and starts.dtype is _i32 and starts.get_device() == at and starts.is_contiguous()
            and (context_lens is None or (context_lens.numel() == B and context_lens.dtype is _i32
                                          and context_lens.get_device() == at and context_lens.is_contiguous()))
            and K.numel() == size and V.numel() == size and K.dtype is _f32 and V.dtype is _f32 and K.get_device() == at
            and V.get_device() == at and K.is_contiguous() and V.is_contiguous()):
        _refuse("kv8_cache_read", starts, *(() if context_lens is None else (context_lens,)), K, V)
    k, v, ks, vs = cache
    st = _fns["ie_kv8_cache_read"](
        B, n, starts.data_ptr(), None if context_lens is None else context_lens.data_ptr(), k.data_ptr(), v.data_ptr(),
        ks.data_ptr(), vs.data_ptr(), block_table.data_ptr(), nbps, H, d, bs, K.data_ptr(), V.data_ptr(),
        _raw_stream_of(at) if stream is None else stream.cuda_stream)
    if st:
        _failed("ie_kv8_cache_read", st)
    return K, V


def decode_kv8_num_splits(B, H_q, H_kv, d, max_ctx, splits=0):
    return call("ie_decode_kv8_num_splits", B, H_q, H_kv, d, max_ctx, splits)


def decode_attn_kv8(Q, cache, block_table, context_lens, max_ctx, splits=0, out=None, workspace=None, stream=None):
    """Q [B, H_q, d] fp32, one token a sequence, over the first context_lens[b]
    <= max_ctx cached positions; returns O [B, H_q, d]."""
    H, bs, d, at, rows, nbps = _kv8("decode_attn_kv8", cache, block_table)
    B, H_q, dq = Q.shape
    if not -0x80000000 <= max_ctx <= 0x7FFFFFFF:
        _past_int("decode_attn_kv8", "max_ctx", max_ctx)
    if out is None:
        out = _new(stream, (B, H_q, d), _f32, Q.device)
    if not (dq == d and rows == B and context_lens.numel() == B and out.numel() == B * H_q * d
            and Q.dtype is _f32 and out.dtype is _f32 and context_lens.dtype is _i32 and Q.get_device() == at
            and out.get_device() == at and context_lens.get_device() == at and Q.is_contiguous() and out.is_contiguous()
            and context_lens.is_contiguous()):
        _refuse("decode_attn_kv8", Q, out, context_lens, block_table)
    if workspace is None:
        S = decode_kv8_num_splits(B, H_q, H, d, max_ctx, splits)
        if S > 1:
            workspace = _new(stream, B * H_q * S * (d + 2), _f32, Q.device)
    elif workspace.dtype is not _f32 or workspace.get_device() != at or not workspace.is_contiguous():
        _refuse("decode_attn_kv8", workspace)
    k, v, ks, vs = cache
    st = _fns["ie_decode_attn_kv8"](
        B, H_q, H, d, Q.data_ptr(), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), block_table.data_ptr(),
        context_lens.data_ptr(), max_ctx, bs, nbps, out.data_ptr(), None if workspace is None else workspace.data_ptr(),
        0 if workspace is None else 4 * workspace.numel(), splits,
        _raw_stream_of(at) if stream is None else stream.cuda_stream)
    if st:
        _failed("ie_decode_attn_kv8", st)
    return out


def prefill_attn_kv8(Q, cache, block_table, start_pos, out=None, workspace=None, stream=None):
    """Q [B, P, H_q, d] fp32, token t at position start_pos + t with its rows
    cached; returns causal O [B, P, H_q, d].  workspace: fp32, at least
    ie_prefill_kv8_workspace_bytes (made here where the call has use for one)."""
    H, bs, d, at, rows, nbps = _kv8("prefill_attn_kv8", cache, block_table)
    B, P, H_q, dq = Q.shape
    if not -0x80000000 <= start_pos <= 0x7FFFFFFF:
        _past_int("prefill_attn_kv8", "start_pos", start_pos)
    if out is None:
        out = _new(stream, (B, P, H_q, d), _f32, Q.device)
    if not (dq == d and rows == B and out.numel() == B * P * H_q * d and Q.dtype is _f32 and out.dtype is _f32
            and Q.get_device() == at and out.get_device() == at and Q.is_contiguous() and out.is_contiguous()):
        _refuse("prefill_attn_kv8", Q, out, block_table)
    if workspace is None:
        need = _fns["ie_prefill_kv8_workspace_bytes"](B, P, H_q, H, d, start_pos)
        if need:
            workspace = _new(stream, need // 4, _f32, Q.device)
    elif workspace.dtype is not _f32 or workspace.get_device() != at or not workspace.is_contiguous():
        _refuse("prefill_attn_kv8", workspace)
    k, v, ks, vs = cache
    st = _fns["ie_prefill_attn_kv8"](
        B, P, H_q, H, d, Q.data_ptr(), k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), block_table.data_ptr(),
        nbps, bs, start_pos, out.data_ptr(), None if workspace is None else workspace.data_ptr(),
        0 if workspace is None else 4 * workspace.numel(), _raw_stream_of(at) if stream is None else stream.cuda_stream)
    if st:
        _failed("ie_prefill_attn_kv8", st)
    return out


class TokenLogprobs(NamedTuple):
    """What token_logprobs returns, one entry per row; top_* are [rows, k]."""
    logprobs: "torch.Tensor"  # noqa: F821
    ranks: "torch.Tensor"  # noqa: F821
    entropy: "torch.Tensor"  # noqa: F821
    top_logprobs: "torch.Tensor"  # noqa: F821
    top_indices: "torch.Tensor"  # noqa: F821


def token_logprobs(logits, targets=None, k=0, out=None, workspace=None, stream=None):
    """Log probability and rank of targets[r] (int32, -1: none) under row r of
    logits [rows, n] fp32 (rows may lie apart), the row's entropy, and its k
    most likely tokens with their log probabilities (include/ie_logprobs.h)."""
    if _device_index is None:
        _bind_torch()
    rows, n = logits.shape
    at = _device_index()
    ld, step = logits.stride()
    if (logits.get_device() != at or logits.dtype is not _f32 or (n > 1 and step != 1)
            or (rows > 1 and not n <= ld <= 0x7FFFFFFF)):
        raise ValueError(f"token_logprobs: logits need to be fp32 rows on cuda:{at}, got {logits.dtype} strides "
                         f"{(ld, step)} on {logits.device}")
    if targets is not None and not (targets.numel() == rows and targets.dtype is _i32 and targets.get_device() == at
                                    and targets.is_contiguous()):
        _refuse("token_logprobs", targets)
    if out is None:
        dev = logits.device
        out = (_new(stream, rows, _f32, dev), _new(stream, rows, _i32, dev), _new(stream, rows, _f32, dev),
               _new(stream, (rows, k), _f32, dev), _new(stream, (rows, k), _i32, dev))
        lp, rk, en, tv, ti = out
    else:
        lp, rk, en, tv, ti = out
        if not (lp.numel() == rows and rk.numel() == rows and en.numel() == rows and tv.numel() == rows * k
                and ti.numel() == rows * k and lp.dtype is _f32 and rk.dtype is _i32 and en.dtype is _f32
                and tv.dtype is _f32 and ti.dtype is _i32 and lp.get_device() == at and rk.get_device() == at
                and en.get_device() == at and tv.get_device() == at and ti.get_device() == at and lp.is_contiguous()
                and rk.is_contiguous() and en.is_contiguous() and tv.is_contiguous() and ti.is_contiguous()):
            _refuse("token_logprobs", lp, rk, en, tv, ti)
    if workspace is None:
        need = _fns["ie_token_logprobs_workspace_bytes"](rows, n, k)
        if need:
            workspace = _new(stream, need // 4, _f32, logits.device)
    elif workspace.dtype is not _f32 or workspace.get_device() != at or not workspace.is_contiguous():
        _refuse("token_logprobs", workspace)
    st = _fns["ie_token_logprobs"](
        rows, logits.data_ptr(), ld if rows > 1 else n, n, None if targets is None else targets.data_ptr(), k, lp.data_ptr(),
        rk.data_ptr(), en.data_ptr(), tv.data_ptr(), ti.data_ptr(), None if workspace is None else workspace.data_ptr(),
        0 if workspace is None else 4 * workspace.numel(), _raw_stream_of(at) if stream is None else stream.cuda_stream)
    if st:
        _failed("ie_token_logprobs", st)
    return TokenLogprobs(lp, rk, en, tv, ti)


# ---------------------------------------------------------------- engine
GPT2_SMALL = dict(n_layers=12, n_heads=12, d_model=768, d_ff=3072, vocab_size=50257, max_seq_len=1024)


def write_random_model(path, seed=0, **cfg):
    c = dict(GPT2_SMALL, **cfg)
    check("ie_engine_write_random_model", str(path).encode(), c["n_layers"], c["n_heads"], c["d_model"],
          c["d_ff"], c["vocab_size"], c["max_seq_len"], seed)


class Engine:
    """GPT-2 decode engine (include/ie_engine.h).  model_dir=None builds a
    random model of the given shape (GPT-2 Small by default).  kv_dtype: KV_F32,
    KV_BF16 or KV_I8 (the 8-bit cache of include/ie_kv8.h)."""

    def __init__(self, model_dir=None, seed=0, max_batch=1, kv_dtype=KV_F32, int8_lm_head=False,
                 use_graph=True, fuse=True, prefill=True, prefill_chunk=0, backend=BACKEND_INT8, **cfg):
        import numpy as np  # noqa: F401

        c = dict(GPT2_SMALL, **cfg)
        h = ctypes.c_void_p()
        check("ie_engine_create", ctypes.byref(h), None if model_dir is None else str(model_dir).encode(),
              c["n_layers"], c["n_heads"], c["d_model"], c["d_ff"], c["vocab_size"], c["max_seq_len"], seed,
              max_batch, kv_dtype, int(int8_lm_head), int(use_graph), int(fuse), int(prefill), prefill_chunk,
              backend)
        self.h = h
        v = (ctypes.c_int * 7)()
        check("ie_engine_config", h, ctypes.cast(v, ctypes.c_void_p))
        self.cfg = dict(zip(("n_layers", "n_heads", "d_model", "d_ff", "vocab_size", "max_seq_len", "d_head"),
                            list(v)))

    def close(self):
        if getattr(self, "h", None):
            load().ie_engine_destroy(self.h)
            self.h = None

    __del__ = close

    def reset(self):
        check("ie_engine_reset", self.h)

    def step(self, tokens, want_logits=True):
        import numpy as np

        toks = np.ascontiguousarray(tokens, dtype=np.int32)
        B = toks.shape[0]
        V = self.cfg["vocab_size"]
        logits = np.empty((B, V), dtype=np.float32) if want_logits else None
        check("ie_engine_step", self.h, B, toks.ctypes.data_as(ctypes.c_void_p),
              None if logits is None else logits.ctypes.data_as(ctypes.c_void_p), None)
        return logits

    def prefill(self, tokens, want_logits=True):
        """tokens [B, P] at the current position -> last-token logits [B, V]."""
        import numpy as np

        toks = np.ascontiguousarray(tokens, dtype=np.int32)
        B, P = toks.shape
        logits = np.empty((B, self.cfg["vocab_size"]), dtype=np.float32) if want_logits else None
        check("ie_engine_prefill", self.h, B, P, toks.ctypes.data_as(ctypes.c_void_p),
              None if logits is None else logits.ctypes.data_as(ctypes.c_void_p), None)
        return logits

    def score(self, tokens, k=0):
        """tokens [B, P] at the current position (a prefill) -> TokenLogprobs of numpy
        arrays [B, P] and [B, P, k]: entry [b, t] is the log probability of
        tokens[b, t + 1] after the ones before it, its rank, and that prediction's
        entropy and k most likely tokens; the last entry has no token to score."""
        import numpy as np

        toks = np.ascontiguousarray(tokens, dtype=np.int32)
        B, P = toks.shape
        out = (np.zeros((B, P), np.float32), np.zeros((B, P), np.int32), np.zeros((B, P), np.float32),
               np.zeros((B, P, max(k, 0)), np.float32), np.zeros((B, P, max(k, 0)), np.int32))
        check("ie_engine_score", self.h, B, P, toks.ctypes.data, k, *(a.ctypes.data for a in out))
        return TokenLogprobs(*out)

    def generate(self, prompts, max_new, ignore_eos=False):
        """prompts [B, P] int -> (tokens [B, max_new] with -1 padding, metrics dict)."""
        import numpy as np

        p = np.ascontiguousarray(prompts, dtype=np.int32)
        B, P = p.shape
        out = np.full((B, max_new), -1, dtype=np.int32)
        m = Metrics()
        check("ie_engine_generate", self.h, B, P, p.ctypes.data_as(ctypes.c_void_p), max_new, int(ignore_eos),
              out.ctypes.data_as(ctypes.c_void_p), ctypes.byref(m))
        return out, m.as_dict()

    def generate_one(self, prompt, max_new, temperature=0.8, top_k=40, greedy=False, reset=True):
        """GPT2Engine::generate for one prompt -> (generated ids, metrics dict)."""
        import numpy as np

        p = np.ascontiguousarray(prompt, dtype=np.int32).reshape(-1)
        out = np.full(max_new, -1, dtype=np.int32)
        n = ctypes.c_int(0)
        m = Metrics()
        check("ie_engine_generate_one", self.h, len(p), p.ctypes.data_as(ctypes.c_void_p), max_new,
              ctypes.c_float(temperature), top_k, int(greedy), int(reset), out.ctypes.data_as(ctypes.c_void_p),
              ctypes.byref(n), ctypes.byref(m))
        return out[: n.value].tolist(), m.as_dict()

    def generate_text(self, tokenizer, prompt, max_new, temperature=0.8, top_k=40, greedy=False, reset=True):
        """The reference's text path (src/main.cpp:224-230, 360-367): the prompt
        encoded by the BPE tokenizer, GPT2Engine::generate, the ids decoded ->
        (generated bytes, generated ids, metrics dict)."""
        ids = tokenizer.encode(prompt)
        if not ids:
            raise ValueError("the prompt encodes to no tokens")
        toks, m = self.generate_one(ids, max_new, temperature, top_k, greedy, reset)
        return tokenizer.decode(toks), toks, m

    def session_tokens(self):
        return load().ie_engine_session_tokens(self.h)

    def step_bytes(self, batch):
        return load().ie_engine_step_bytes(self.h, batch)


class Tokenizer:
    """GPT-2 byte-level BPE tokenizer (include/ie_tokenizer.h), the reference's
    BPETokenizer (include/tokenizer.h:7-25): vocab.json and merges.txt from
    model_dir.  encode takes str or bytes; decode returns bytes, since a token
    can end inside a multi-byte character."""

    def __init__(self, model_dir):
        h = ctypes.c_void_p()
        check("ie_tokenizer_create", ctypes.byref(h), os.fsencode(model_dir))
        self.h = h

    def close(self):
        if self.h:
            load().ie_tokenizer_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def encode(self, text):
        b = text.encode("utf-8") if isinstance(text, str) else bytes(text)
        n = ctypes.c_size_t()
        check("ie_tokenizer_encode", self.h, b, len(b), None, 0, ctypes.byref(n))
        out = (ctypes.c_int * max(n.value, 1))()
        check("ie_tokenizer_encode", self.h, b, len(b), out, n.value, ctypes.byref(n))
        return list(out[:n.value])

    def decode(self, ids):
        ids = [int(i) for i in ([ids] if isinstance(ids, numbers.Integral) else ids)]
        arr = (ctypes.c_int * max(len(ids), 1))(*ids)
        n = ctypes.c_size_t()
        check("ie_tokenizer_decode", self.h, arr, len(ids), None, 0, ctypes.byref(n))
        buf = ctypes.create_string_buffer(max(n.value, 1))
        check("ie_tokenizer_decode", self.h, arr, len(ids), buf, n.value, ctypes.byref(n))
        return buf.raw[:n.value]

    @property
    def vocab_size(self):
        return load().ie_tokenizer_vocab_size(self.h)

    @property
    def eos_token(self):
        return load().ie_tokenizer_eos_token(self.h)
