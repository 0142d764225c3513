"""neonengine_amd -- ctypes view of the gfx950 gpt-oss token-loop library.

The product is libneon_gptoss.so (hand-written HIP kernels for gfx950 behind
the C-ABI in include/neon_gptoss.h).  This module binds that ABI for Python
callers (tests, bench.py): every call goes straight into the shared library;
there is no Python or CPU fallback, and loading fails loudly when the library
has not been built.

Device memory for the kernel-level entry points comes from torch tensors on
``cuda`` (HIP) devices; only their data pointers cross the boundary.
"""
from __future__ import annotations

import ctypes as C
import os

HERE = os.path.dirname(os.path.abspath(__file__))
# NEON_GPTOSS_LIB selects another build of the library (e.g. the host-
# sanitizer build neonengine_amd/_asan/libneon_gptoss.so)
LIB_PATH = os.environ.get("NEON_GPTOSS_LIB") or os.path.join(HERE, "libneon_gptoss.so")

NEON_OK, NEON_EINVAL, NEON_ENOMEM, NEON_EHIP = 0, 1, 2, 3
NEON_ENAN_SCALE, NEON_EKV_FULL, NEON_ERANGE_TOKEN, NEON_ESTATE = 4, 5, 6, 7
STATUS_NAMES = {0: "NEON_OK", 1: "NEON_EINVAL", 2: "NEON_ENOMEM", 3: "NEON_EHIP",
                4: "NEON_ENAN_SCALE", 5: "NEON_EKV_FULL", 6: "NEON_ERANGE_TOKEN",
                7: "NEON_ESTATE"}

# Every symbol include/neon_gptoss.h declares (tests check the exports).
EXPORTS = (
    "neon_config_preset", "neon_ctx_create", "neon_ctx_destroy", "neon_last_error",
    "neon_init_random", "neon_load_tensor", "neon_prefill", "neon_decode",
    "neon_read_tokens", "neon_read_logits", "neon_read_activation", "neon_seq_len",
    "neon_tensor_ptr",
    "neon_mxfp4_dequant", "neon_mxfp4_gemv", "neon_gemv_bf16", "neon_rmsnorm",
    "neon_rope_yarn", "neon_router_topk", "neon_moe_layer", "neon_moe_experts",
    "neon_attn_decode", "neon_set_prefill_mode", "neon_gemm_bf16", "neon_moe_prefill",
    "neon_attn_prefill", "neon_set_sampling", "neon_sample", "neon_set_decode_mode",
    "neon_gemv_bf16_mfma", "neon_device_check", "neon_moe_layer_noalloc",
    "neon_prefill_ragged", "neon_seq_lens", "neon_moe_prefill_mx8", "neon_mx8_quant",
    "neon_rope_table", "neon_moe_layer_workspace", "neon_attn_decode_workspace",
    "neon_attn_decode_counters", "neon_sample_workspace", "neon_moe_prefill_workspace",
    "neon_seq_add", "neon_seq_remove",
    "neon_paged_append", "neon_paged_gather", "neon_paged_attn", "neon_paged_attn_workspace",
    "neon_paged_attn_counters", "neon_sample_rows", "neon_sample_rows_workspace",
    "neon_beam_select", "neon_beam_select_workspace", "neon_beam_reorder", "neon_pages_fork",
    "neon_pages_workspace", "neon_pages_counters", "neon_pages_copy", "neon_pages_compact",
)


class NeonError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"{STATUS_NAMES.get(status, status)}: {msg}")
        self.status = status


class Config(C.Structure):
    _fields_ = [(n, C.c_int32) for n in (
        "n_layers", "hidden", "n_heads", "n_kv_heads", "head_dim",
        "n_experts", "top_k", "intermediate", "vocab",
        "sliding_window", "max_seq", "max_batch")] + [
        (n, C.c_float) for n in ("rope_theta", "rope_factor", "rope_beta_fast", "rope_beta_slow")] + [
        ("rope_orig_max_pos", C.c_int32)] + [
        (n, C.c_float) for n in ("rms_eps", "swiglu_limit", "swiglu_alpha")]

    def as_dict(self):
        return {n: getattr(self, n) for n, _ in self._fields_}


class PagedKVStruct(C.Structure):
    """neon_paged_kv."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scales", C.c_void_p),
                ("v_scales", C.c_void_p)] + [(n, C.c_int32) for n in (
                    "format", "n_pages", "page_size", "n_kv_heads", "head_dim")]


_lib = None
_P, _I, _I64, _U64, _F, _SZ = C.c_void_p, C.c_int, C.c_int64, C.c_uint64, C.c_float, C.c_size_t


def lib():
    """Load libneon_gptoss.so (raises if it is not built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -m neonengine_amd._build` "
                "(the gfx950 HIP library is required; there is no fallback)")
        # One HIP runtime per process: torch bundles its own libamdhip64 (same
        # soname, libamdhip64.so.7), and a process that loads /opt/rocm's copy
        # through this library first and torch's afterwards holds two runtimes,
        # of which ours then sees no device.  Loading torch first makes the
        # library's libamdhip64.so.7 dependency resolve to torch's copy.
        try:
            import torch  # noqa: F401
        except ImportError:
            pass
        L = C.CDLL(LIB_PATH)
        sig = {
            "neon_config_preset": [C.c_char_p, _P],
            "neon_ctx_create": [_P, _I, _P],
            "neon_ctx_destroy": [_P],
            "neon_last_error": [_P],
            "neon_init_random": [_P, _U64, _P],
            "neon_load_tensor": [_P, C.c_char_p, _P, _SZ],
            "neon_prefill": [_P, _P, _I, _I, _P],
            "neon_prefill_ragged": [_P, _P, _P, _I, _P],
            "neon_decode": [_P, _I, _P],
            "neon_read_tokens": [_P, _I, _I, _P, _P],
            "neon_read_logits": [_P, _P, _P],
            "neon_read_activation": [_P, C.c_char_p, _P, _SZ, _P],
            "neon_seq_len": [_P, _P],
            "neon_seq_lens": [_P, _P],
            "neon_seq_add": [_P, _P, _I, _P, _P],
            "neon_seq_remove": [_P, _I, _P],
            "neon_tensor_ptr": [_P, C.c_char_p, _P, _P],
            "neon_mxfp4_dequant": [_P, _P, _I64, _P, _P],
            "neon_mxfp4_gemv": [_P, _P, _P, _P, _P, _I, _I, _I, _P],
            "neon_gemv_bf16": [_P, _P, _P, _P, _I, _I, _I, _P],
            "neon_rmsnorm": [_P, _P, _P, _I, _I, _F, _P],
            "neon_rope_table": [_P, _I, _P, _P],
            "neon_rope_yarn": [_P, _P, _I, _I, _I, _P, _I, _P],
            "neon_router_topk": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P],
            "neon_moe_layer": [_P] * 13 + [_I] * 5 + [_F, _F, _P, _SZ, _P],
            "neon_moe_experts": [_P] * 12 + [_I] * 5 + [_F, _F, _P],
            "neon_attn_decode": [_P] * 6 + [_I] * 6 + [_P, _SZ, _P, _SZ, _P],
            "neon_set_prefill_mode": [_P, _I],
            "neon_gemm_bf16": [_P] * 4 + [_I] * 4 + [_P],
            "neon_moe_prefill": [_P] * 10 + [_I] * 5 + [_F, _F, _P, _SZ, _P],
            "neon_moe_prefill_mx8": [_P] * 10 + [_I] * 5 + [_F, _F, _P, _SZ, _P],
            "neon_mx8_quant": [_P, _I64, _I, _P, _P, _P, _P, _P],
            "neon_attn_prefill": [_P] * 5 + [_I] * 6 + [_P],
            "neon_set_sampling": [_P, _F, _F, _U64],
            "neon_sample": [_P, _I, _I, _F, _F, _U64, _P, _P, _P, _SZ, _P],
            "neon_set_decode_mode": [_P, _I],
            "neon_gemv_bf16_mfma": [_P, _P, _P, _P, _I, _I, _I, _P],
            "neon_device_check": [_P],
            "neon_moe_layer_noalloc": [_P] * 13 + [_I] * 5 + [_F, _F, _P],
            "neon_paged_append": [_P, _P, _I64, _P, _I, _P, _P, _P, _I, _P, _I, _I, _I, _P],
            "neon_paged_gather": [_P, _P, _P, _P, _I, _P, _P, _I, _I, _P],
            "neon_paged_attn": [_P, _P, _I64, _P, _P, _P, _P, _I, _P] + [_I] * 4 +
                               [_P, _SZ, _P, _SZ, _P],
            "neon_sample_rows": [_P, _I64, _I, _I] + [_P] * 7 + [_SZ, _P],
            "neon_beam_select": [_P, _I64, _I, _I, _I, _P, _P, _I] + [_P] * 7 + [_SZ, _P],
            "neon_beam_reorder": [_P] + [_I] * 6 + [_P] * 3,
            "neon_pages_fork": [_P] * 3 + [_I] + [_P] * 9 + [_I] * 4 + [_P, _SZ, _P, _SZ, _P],
            "neon_pages_copy": [_P, _I, _P, _P, _P, _I, _P],
            "neon_pages_compact": [_P] * 8 + [_I] * 4 + [_P, _SZ, _P],
        }
        for name, args in sig.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = C.c_int
        # workspace-size queries (size_t results)
        for name, args in {"neon_moe_layer_workspace": [_I] * 4,
                           "neon_attn_decode_workspace": [_I] * 6,
                           "neon_attn_decode_counters": [_I] * 2,
                           "neon_sample_workspace": [_I] * 2,
                           "neon_moe_prefill_workspace": [_I] * 6,
                           "neon_paged_attn_workspace": [_I] * 5,
                           "neon_paged_attn_counters": [_I] * 5,
                           "neon_sample_rows_workspace": [_I] * 2,
                           "neon_beam_select_workspace": [_I] * 4,
                           "neon_pages_workspace": [_I] * 2,
                           "neon_pages_counters": [_I]}.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = _SZ
        L.neon_ctx_destroy.restype = None
        L.neon_last_error.restype = C.c_char_p
        _lib = L
    return _lib


def _check(status: int, ctx=None):
    if status != NEON_OK:
        msg = lib().neon_last_error(ctx)
        raise NeonError(status, msg.decode() if msg else "")


def device_check(stream=None):
    """Synchronise and raise NeonError(NEON_EINVAL) if a kernel-level call on
    the current device saw an input out of range (an expert id outside [0, E); row
    starts, lengths, page ids, sampling parameters, scores, parents or reference counts)
    since the last check, NeonError(NEON_EKV_FULL) if pages ran out."""
    _check(lib().neon_device_check(stream))


def config_preset(name: str = "gpt-oss-20b", **overrides) -> Config:
    cfg = Config()
    _check(lib().neon_config_preset(name.encode(), C.byref(cfg)))
    for k, v in overrides.items():
        setattr(cfg, k, v)
    return cfg


# The smallest calls are bound by this file: an attention step over a window is a
# 5.2 us kernel under a 10.5 us wrapper when each pointer is boxed, the device
# looked for and the workspace sized on every call, and 9.2 us as it stands.
# Every entry point has its argtypes, so a plain int passes as a pointer whole.
def _ptr(t):
    """Device pointer of a torch tensor (None -> NULL)."""
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        if not t.is_contiguous():
            raise ValueError("tensor must be contiguous")
        return t.data_ptr()
    return C.c_void_p(int(t))


def _nbytes(t):
    """Size in bytes of a torch tensor (None -> 0)."""
    if t is None:
        return 0
    return t.numel() * t.element_size()


_current = None  # (device index, its stream's handle) functions, once a device was
                 # found (a process does not lose it again)
_fp16 = None     # torch.float16 from then on: it has the size of bf16
_int32 = _float32 = None  # torch's


def _find_current():
    """Functions that give torch's current device, and its current stream there:
    torch's own shortcuts to the bare numbers where it has them
    (torch.cuda.current_stream() makes an object for 3 us)."""
    global _current, _fp16, _int32, _float32
    import torch
    _fp16, _int32, _float32 = torch.float16, torch.int32, torch.float32
    if not torch.cuda.is_available():
        return None
    torch.cuda.init()
    try:
        from torch._C import _cuda_getCurrentRawStream as raw, _cuda_getDevice as device
        raw(device())
        _current = (device, raw)
    except Exception:
        _current = (torch.cuda.current_device, lambda d: torch.cuda.current_stream(d).cuda_stream)
    return _current


def _stream(stream):
    """Stream handle (None -> torch's current stream, or the default one)."""
    if stream is None:
        try:
            c = _current or _find_current()
            return c[1](c[0]()) if c else None
        except Exception:
            return None
    if hasattr(stream, "cuda_stream"):
        return C.c_void_p(stream.cuda_stream)
    return C.c_void_p(int(stream))


# ---------------------------------------------------------------------------
# kernel-level entry points (torch tensors on the HIP device; bf16 tensors may
# be torch.bfloat16 or int16/uint16 views of the bit patterns)
# ---------------------------------------------------------------------------
def mxfp4_dequant(codes, scales, out, stream=None):
    _check(lib().neon_mxfp4_dequant(_ptr(codes), _ptr(scales), scales.numel(), _ptr(out),
                                    _stream(stream)))


def mxfp4_gemv(codes, scales, bias, x, y, N, K, B, stream=None):
    _check(lib().neon_mxfp4_gemv(_ptr(codes), _ptr(scales), _ptr(bias), _ptr(x), _ptr(y),
                                 N, K, B, _stream(stream)))


def gemv_bf16(W, bias, x, y, N, K, B, stream=None):
    _check(lib().neon_gemv_bf16(_ptr(W), _ptr(bias), _ptr(x), _ptr(y), N, K, B,
                                _stream(stream)))


def gemv_bf16_mfma(W, bias, x, y, N, K, B, stream=None):
    _check(lib().neon_gemv_bf16_mfma(_ptr(W), _ptr(bias), _ptr(x), _ptr(y), N, K, B,
                                     _stream(stream)))


def rmsnorm(x, w, out, B, H, eps=1e-5, stream=None):
    _check(lib().neon_rmsnorm(_ptr(x), _ptr(w), _ptr(out), B, H, eps, _stream(stream)))


def rope_table(cfg: Config, n_pos, table, stream=None):
    """table: device fp32 [2][n_pos][head_dim / 2] (cos, then sin)."""
    _check(lib().neon_rope_table(C.byref(cfg), n_pos, _ptr(table), _stream(stream)))


def rope_yarn(x, pos, n_tok, n_heads, head_dim, table, n_pos, stream=None):
    _check(lib().neon_rope_yarn(_ptr(x), _ptr(pos), n_tok, n_heads, head_dim, _ptr(table),
                                n_pos, _stream(stream)))


def _workspace(nbytes, zero=False):
    """A caller-side device buffer of nbytes (torch), for callers that do not
    keep their own workspace; the library itself allocates nothing."""
    import torch
    n = max(int(nbytes), 1)
    return torch.zeros(n, dtype=torch.uint8, device="cuda") if zero else \
        torch.empty(n, dtype=torch.uint8, device="cuda")


def router_topk(x, W, b, idx, score, logits, B, E, H, k, stream=None):
    if logits is None:  # the C-ABI takes the logits buffer from the caller
        logits = _workspace(B * E * 4)
    _check(lib().neon_router_topk(_ptr(x), _ptr(W), _ptr(b), _ptr(idx), _ptr(score),
                                  _ptr(logits), B, E, H, k, _stream(stream)))


def moe_layer_workspace(B, E, I, k):
    return lib().neon_moe_layer_workspace(B, E, I, k)


def moe_layer(x, router_w, router_b, gu_codes, gu_scales, gu_bias, dn_codes, dn_scales,
              dn_bias, residual, out, idx, score, B, E, H, I, k, alpha=1.702, limit=7.0,
              stream=None, workspace=None):
    if workspace is None:
        workspace = _workspace(moe_layer_workspace(B, E, I, k))
    _check(lib().neon_moe_layer(
        _ptr(x), _ptr(router_w), _ptr(router_b), _ptr(gu_codes), _ptr(gu_scales),
        _ptr(gu_bias), _ptr(dn_codes), _ptr(dn_scales), _ptr(dn_bias), _ptr(residual),
        _ptr(out), _ptr(idx), _ptr(score), B, E, H, I, k, alpha, limit, _ptr(workspace),
        _nbytes(workspace), _stream(stream)))


def moe_layer_noalloc(x, router_w, router_b, gu_codes, gu_scales, gu_bias, dn_codes,
                      dn_scales, dn_bias, residual, out, idx, score, B, E, H, I, k,
                      alpha=1.702, limit=7.0, stream=None):
    """neon_moe_layer with its scratch in the library's fixed per-GPU array
    (no allocation; overlapping calls on one GPU race)."""
    _check(lib().neon_moe_layer_noalloc(
        _ptr(x), _ptr(router_w), _ptr(router_b), _ptr(gu_codes), _ptr(gu_scales),
        _ptr(gu_bias), _ptr(dn_codes), _ptr(dn_scales), _ptr(dn_bias), _ptr(residual),
        _ptr(out), _ptr(idx), _ptr(score), B, E, H, I, k, alpha, limit, _stream(stream)))


def moe_experts(x, idx, score, gu_codes, gu_scales, gu_bias, dn_codes, dn_scales, dn_bias,
                residual, out, act, B, E, H, I, k, alpha=1.702, limit=7.0, stream=None):
    _check(lib().neon_moe_experts(
        _ptr(x), _ptr(idx), _ptr(score), _ptr(gu_codes), _ptr(gu_scales), _ptr(gu_bias),
        _ptr(dn_codes), _ptr(dn_scales), _ptr(dn_bias), _ptr(residual), _ptr(out), _ptr(act),
        B, E, H, I, k, alpha, limit, _stream(stream)))


def attn_decode_workspace(B, Hq, Hkv, D, T_max, window):
    """(workspace bytes, counter bytes) of neon_attn_decode."""
    L = lib()
    return (L.neon_attn_decode_workspace(B, Hq, Hkv, D, T_max, window),
            L.neon_attn_decode_counters(B, Hkv))


def attn_decode(q, k_cache, v_cache, sinks, pos, out, B, Hq, Hkv, D, T_max, window,
                stream=None, workspace=None, counters=None):
    """counters: zero-filled once by the caller (each call leaves it zero)."""
    if workspace is None or counters is None:
        wb, cb = attn_decode_workspace(B, Hq, Hkv, D, T_max, window)
        if workspace is None and wb:
            workspace = _workspace(wb)
        if counters is None:
            counters = _workspace(cb, zero=True)
    _check(lib().neon_attn_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(sinks),
                                  _ptr(pos), _ptr(out), B, Hq, Hkv, D, T_max, window,
                                  _ptr(workspace), _nbytes(workspace), _ptr(counters),
                                  _nbytes(counters), _stream(stream)))


def gemm_bf16(A, W, bias, C_, M, N, K, accumulate=False, stream=None):
    _check(lib().neon_gemm_bf16(_ptr(A), _ptr(W), _ptr(bias), _ptr(C_), M, N, K,
                                1 if accumulate else 0, _stream(stream)))


def moe_prefill_workspace(M, E, H, I, k, mx8=False):
    return lib().neon_moe_prefill_workspace(M, E, H, I, k, 1 if mx8 else 0)


def moe_prefill(x, idx, score, gu_codes, gu_scales, gu_bias, dn_codes, dn_scales, dn_bias,
                h, M, E, H, I, k, alpha=1.702, limit=7.0, stream=None, workspace=None):
    if workspace is None:
        workspace = _workspace(moe_prefill_workspace(M, E, H, I, k))
    _check(lib().neon_moe_prefill(
        _ptr(x), _ptr(idx), _ptr(score), _ptr(gu_codes), _ptr(gu_scales), _ptr(gu_bias),
        _ptr(dn_codes), _ptr(dn_scales), _ptr(dn_bias), _ptr(h), M, E, H, I, k, alpha, limit,
        _ptr(workspace), _nbytes(workspace), _stream(stream)))


def moe_prefill_mx8(x, idx, score, gu_codes, gu_scales, gu_bias, dn_codes, dn_scales, dn_bias,
                    h, M, E, H, I, k, alpha=1.702, limit=7.0, stream=None, workspace=None):
    if workspace is None:
        workspace = _workspace(moe_prefill_workspace(M, E, H, I, k, mx8=True))
    _check(lib().neon_moe_prefill_mx8(
        _ptr(x), _ptr(idx), _ptr(score), _ptr(gu_codes), _ptr(gu_scales), _ptr(gu_bias),
        _ptr(dn_codes), _ptr(dn_scales), _ptr(dn_bias), _ptr(h), M, E, H, I, k, alpha, limit,
        _ptr(workspace), _nbytes(workspace), _stream(stream)))


def mx8_quant(x, rows, K, hi, lo, s_hi, s_lo, stream=None):
    _check(lib().neon_mx8_quant(_ptr(x), rows, K, _ptr(hi), _ptr(lo), _ptr(s_hi), _ptr(s_lo),
                                _stream(stream)))


def attn_prefill(q, k_cache, v_cache, sinks, out, M, Hq, Hkv, D, T_max, window, stream=None):
    _check(lib().neon_attn_prefill(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(sinks),
                                   _ptr(out), M, Hq, Hkv, D, T_max, window, _stream(stream)))


def sample_workspace(B, V):
    return lib().neon_sample_workspace(B, V)


def sample_logits(logits, B, V, temperature, top_p, seed, pos, out_ids, stream=None,
                  workspace=None):
    if workspace is None:
        workspace = _workspace(sample_workspace(B, V))
    _check(lib().neon_sample(_ptr(logits), B, V, temperature, top_p, seed, _ptr(pos),
                             _ptr(out_ids), _ptr(workspace), _nbytes(workspace),
                             _stream(stream)))


KV_BF16, KV_MXFP4 = 0, 1


class PagedKV:
    """A paged KV cache over the caller's pools (neon_paged_kv).

    k, v: bf16 [n_pages][n_kv_heads][page_size][head_dim]; or, with k_scales
    and v_scales (uint8 [..][head_dim / 32]), MXFP4 codes (uint8 [..][head_dim / 2])."""

    def __init__(self, k, v, k_scales=None, v_scales=None):
        mx = k_scales is not None
        pools = (k, v, k_scales, v_scales) if mx or v_scales is not None else (k, v)
        if any(t is None or t.dim() != 4 for t in pools):
            raise ValueError("PagedKV: pools are [n_pages][n_kv_heads][page_size][..], MXFP4 ones "
                             "with scales for both")
        n_pages, heads, page, width = k.shape
        dim = width * 2 if mx else width
        if tuple(v.shape) != tuple(k.shape) or \
                any(tuple(t.shape) != (n_pages, heads, page, dim // 32) for t in pools[2:]):
            raise ValueError("PagedKV: k, v (and their scales) must have matching shapes")
        import torch
        if any(t.element_size() != (1 if mx else 2) or t.dtype is torch.float16 for t in pools):
            raise ValueError("PagedKV: bf16 pools have 2-byte elements, MXFP4 codes and scales 1")
        self.pools = pools  # keeps them alive
        self.device = k.get_device()
        if any(t.get_device() != self.device for t in pools):
            raise ValueError("PagedKV: pools on one device")
        self.format = KV_MXFP4 if mx else KV_BF16
        self.n_kv_heads, self.head_dim = heads, dim
        self.struct = PagedKVStruct(*(_ptr(t) for t in pools), *(() if mx else (None, None)),
                                    self.format, n_pages, page, heads, dim)
        self.ref = C.addressof(self.struct)


def paged_kv(k, v, k_scales=None, v_scales=None) -> PagedKV:
    return PagedKV(k, v, k_scales, v_scales)


def _arg(t, size, n, name, device, real=None):
    """Device pointer of a contiguous tensor of at least n elements of this size
    on this device (its index), or ValueError: the library trusts the sizes that
    the paged calls derive from other tensors.  real: floating point or not (None:
    bf16, or integers that hold its bits)."""
    if t.element_size() != size or t.numel() < n or t.get_device() != device or \
            not t.is_contiguous() or \
            (t.dtype is _fp16 if real is None else t.is_floating_point() is not real):
        raise ValueError(f"{name}: needs {n} contiguous elements of {size} bytes"
                         f"{' (bf16)' if real is None else ' (floats)' if real else ' (integers)'} on "
                         f"device {device}, has {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.data_ptr()


def _i32(t, n, name, device):
    """_arg of at least n int32: the plans and choices take up to fourteen of these, and
    one test of the type is half of what _arg costs."""
    if t.dtype is not _int32 or t.numel() < n or t.get_device() != device or \
            not t.is_contiguous():
        raise ValueError(f"{name}: needs {n} contiguous int32 on device {device}, has "
                         f"{tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.data_ptr()


def _f32(t, n, name, device):
    """_arg of at least n float32."""
    if t.dtype is not _float32 or t.numel() < n or t.get_device() != device or \
            not t.is_contiguous():
        raise ValueError(f"{name}: needs {n} contiguous float32 on device {device}, has "
                         f"{tuple(t.shape)} of {t.dtype} on {t.device}")
    return t.data_ptr()


def _scratch(nbytes, stream, zero=False):
    """_workspace, allocated (and zeroed) on the stream that the call runs on:
    memory of another one could be in use there still, or handed out again
    before the call is done."""
    if stream is None:
        return _workspace(nbytes, zero)
    import torch
    if not hasattr(stream, "cuda_stream"):
        stream = torch.cuda.ExternalStream(int(stream)) if int(stream) else \
            torch.cuda.default_stream()
    with torch.cuda.stream(stream):
        return _workspace(nbytes, zero)


def _buffer(t, name, device):
    """Device pointer of a contiguous tensor on this device."""
    if t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous memory on device {device}")
    return t.data_ptr()


def _rows(x, size, width, name, device):
    """(device pointer, rows, elements between them) of rows of at least `width`
    elements: contiguous ones, or a slice of wider rows."""
    shape = x.shape
    if x.element_size() != size or x.get_device() != device or len(shape) not in (2, 3) or \
            (x.dtype is _fp16 if size == 2 else not x.is_floating_point()):
        raise ValueError(f"{name}: rows of {'bf16' if size == 2 else 'fp32'} on device {device}")
    n = shape[0]
    has = shape[1] if len(shape) == 2 else shape[1] * shape[2]
    stride = has if has > width else width
    if not x.is_contiguous():
        inner = (1,) if len(shape) == 2 else (shape[2], 1)
        if any(s != w and k > 1 for s, w, k in zip(x.stride()[1:], inner, shape[1:])):
            raise ValueError(f"{name}: each row must be contiguous")
        if n > 1:
            stride = x.stride(0)
    if n and (has < width or stride < width):
        raise ValueError(f"{name}: rows of {width} elements that do not overlap, has {has}, "
                         f"{stride} apart")
    return x.data_ptr(), n, stride


def _on_current(device, stream):
    """The stream's handle (None: the current one); the calls go to the current
    device: tensors elsewhere are refused."""
    c = _current or _find_current()
    if device < 0 or c is None or device != c[0]():
        raise ValueError(f"tensors on device {device}: the call runs on the current HIP device")
    return c[1](device) if stream is None else _stream(stream)


def _batch(kv, q_start, kv_len, page_table, n_rows):
    """(q_start, kv_len, page_table, max_pages, B) of a paged call."""
    device = kv.device
    shape = page_table.shape
    if len(shape) != 2:
        raise ValueError("page_table: [B][max_pages]")
    B, max_pages = shape
    if kv_len.numel() != B:
        raise ValueError("page_table: one row per sequence of kv_len")
    if q_start is not None:
        q_start = _arg(q_start, 4, B + 1, "q_start", device, False)
    elif n_rows != B:
        raise ValueError("without q_start there is one row per sequence")
    return (q_start, _arg(kv_len, 4, B, "kv_len", device, False),
            _arg(page_table, 4, 1, "page_table", device, False), max_pages, B)


def paged_append(kv, qkv, table, q_start, kv_len, page_table, q_out, Hq, stream=None):
    """Rotates q and k of the rows qkv [n_rows][(Hq + 2 n_kv_heads) head_dim]
    and appends k and v to the pages (neon_paged_append).  table: from
    rope_table, fp32 [2][n_pos][head_dim / 2], or None (no rotation)."""
    D, device = kv.head_dim, kv.device
    on = _on_current(device, stream)
    rows, n, stride = _rows(qkv, 2, (Hq + 2 * kv.n_kv_heads) * D, "qkv", device)
    q_start, kv_len, page_table, max_pages, B = _batch(kv, q_start, kv_len, page_table, n)
    q_out = _arg(q_out, 2, n * Hq * D, "q_out", device) if Hq else None
    n_pos = 0
    if table is not None:
        shape = table.shape
        if len(shape) != 3 or shape[0] != 2 or shape[2] != D // 2:
            raise ValueError("table: [2][n_pos][head_dim / 2]")
        n_pos = shape[1]
        table = _arg(table, 4, n_pos * D, "table", device, True)
    _check(lib().neon_paged_append(kv.ref, rows, stride, table, n_pos, q_start, kv_len, page_table,
                                   max_pages, q_out, n, B, Hq, on))


def paged_gather(kv, q_start, kv_len, page_table, k_out, v_out, stream=None):
    """The rows that paged_append writes for the same arguments, as bf16, into
    k_out and v_out [n_rows][n_kv_heads][head_dim] (neon_paged_gather)."""
    n, width, device = k_out.shape[0], kv.n_kv_heads * kv.head_dim, kv.device
    on = _on_current(device, stream)
    q_start, kv_len, page_table, max_pages, B = _batch(kv, q_start, kv_len, page_table, n)
    _check(lib().neon_paged_gather(kv.ref, q_start, kv_len, page_table, max_pages,
                                   _arg(k_out, 2, n * width, "k_out", device),
                                   _arg(v_out, 2, n * width, "v_out", device), n, B, on))


def paged_attn_workspace(n_rows, B, Hq, Hkv, D):
    """(workspace bytes, counter bytes) of neon_paged_attn."""
    L = lib()
    return (L.neon_paged_attn_workspace(n_rows, B, Hq, Hkv, D),
            L.neon_paged_attn_counters(n_rows, B, Hq, Hkv, D))


def paged_attn(kv, q, sinks, q_start, kv_len, page_table, out, Hq, window=0, stream=None,
               workspace=None, counters=None):
    """Attention of the rows q [n_rows][Hq head_dim] over the pages
    (neon_paged_attn).  counters: zero-filled once by the caller (each call
    leaves it zero)."""
    D, device = kv.head_dim, kv.device
    on = _on_current(device, stream)
    rows, n, stride = _rows(q, 2, Hq * D, "q", device)
    q_start, kv_len, page_table, max_pages, B = _batch(kv, q_start, kv_len, page_table, n)
    if sinks is not None:
        sinks = _arg(sinks, 2, Hq, "sinks", device)
    if workspace is None or counters is None:
        wb, cb = paged_attn_workspace(n, B, Hq, kv.n_kv_heads, D)
        if workspace is None:
            workspace = _scratch(wb, stream)
        if counters is None:
            counters = _scratch(cb, stream, zero=True)
    wb, cb = workspace.nbytes, counters.nbytes
    _check(lib().neon_paged_attn(kv.ref, rows, stride, sinks, q_start, kv_len, page_table,
                                 max_pages, _arg(out, 2, n * Hq * D, "out", device), n, B, Hq,
                                 window, _buffer(workspace, "workspace", device), wb,
                                 _buffer(counters, "counters", device), cb, on))


def sample_rows_workspace(B, V):
    return lib().neon_sample_rows_workspace(B, V)


def sample_rows(logits, u, out_ids, temperature=None, top_k=None, top_p=None, min_p=None,
                stream=None, workspace=None):
    """One draw per row of logits [B][V] (fp32; rows may be a slice of wider
    ones) from the random numbers u [B], each parameter a device array [B] or
    None (neon_sample_rows)."""
    if logits.dim() != 2:
        raise ValueError("logits: [B][V]")
    device = logits.get_device()
    on = _on_current(device, stream)
    V = logits.shape[1]
    rows, B, stride = _rows(logits, 4, V, "logits", device)
    if workspace is None:
        workspace = _scratch(sample_rows_workspace(B, V), stream)

    def opt(t, name, real=True):
        return None if t is None else _arg(t, 4, B, name, device, real)

    _check(lib().neon_sample_rows(rows, stride, B, V, opt(temperature, "temperature"),
                                  opt(top_k, "top_k", False), opt(top_p, "top_p"), opt(min_p, "min_p"),
                                  opt(u, "u"), opt(out_ids, "out_ids", False),
                                  _buffer(workspace, "workspace", device), workspace.nbytes, on))


def beam_select_workspace(B, W, V, n_stop):
    return lib().neon_beam_select_workspace(B, W, V, n_stop)


def beam_select(logits, score, W, token, parent, out_score, stop=None, ended=None, stream=None,
                workspace=None):
    """The next beams of requests with W places each (neon_beam_select): logits
    [B W][V] (fp32; rows may be a slice of wider ones), score [B W] fp32; token and
    parent int32, out_score fp32, [B W] each.  stop: int32 ids or None.  ended:
    (end_token, end_parent, end_score) or None."""
    if logits.dim() != 2:
        raise ValueError("logits: [B W][V]")
    device = logits.get_device()
    on = _on_current(device, stream)
    V = logits.shape[1]
    rows, N, stride = _rows(logits, 4, V, "logits", device)
    if W < 1 or N % W:
        raise ValueError(f"logits: {N} rows are not requests of {W} places")
    n_stop = 0 if stop is None else stop.numel()
    if workspace is None:
        workspace = _scratch(beam_select_workspace(N // W, W, V, n_stop), stream)
    end_token = end_parent = end_score = None
    if ended is not None:
        end_token, end_parent, end_score = ended
        end_token = _i32(end_token, N, "end_token", device)
        end_parent = _i32(end_parent, N, "end_parent", device)
        end_score = _f32(end_score, N, "end_score", device)
    _check(lib().neon_beam_select(
        rows, stride, N // W, W, V, _f32(score, N, "score", device),
        _i32(stop, n_stop, "stop", device) if n_stop else None, n_stop,
        _i32(token, N, "token", device), _i32(parent, N, "parent", device),
        _f32(out_score, N, "out_score", device), end_token, end_parent, end_score,
        _buffer(workspace, "workspace", device), workspace.nbytes, on))


class BeamStates:
    """States of beams that move together (neon_beam_reorder): tensors of one shape
    and type, [B W][slabs][T][...], [B W][T][...] or [B W][T]; rows of a multiple of 4
    bytes."""

    def __init__(self, states, W):
        states = tuple(states)
        if not states or W < 1:
            raise ValueError("BeamStates: at least one state and one place")
        shape, size = tuple(states[0].shape), states[0].element_size()
        self.device = states[0].get_device()
        if len(shape) < 2 or shape[0] % W or any(n < 1 for n in shape):
            raise ValueError(f"BeamStates: [B W][slabs][T][..] or [B W][T][..], has {shape}")
        if any(tuple(t.shape) != shape or t.element_size() != size or
               t.get_device() != self.device for t in states):
            raise ValueError("BeamStates: states of one shape and type, on one device")
        starts, nbytes = sorted(t.data_ptr() for t in states), _nbytes(states[0])
        if any(b - a < nbytes for a, b in zip(starts, starts[1:])):
            raise ValueError("BeamStates: two states overlap")
        self.states = states  # keeps them alive
        self.W, self.rows = W, shape[0]
        slabs, T, row = (1, shape[1], shape[2:]) if len(shape) < 4 else (shape[1], shape[2], shape[3:])
        n = size
        for k in row:
            n *= k
        self.ptrs = (C.c_void_p * len(states))(*(_ptr(t) for t in states))
        self.ref = C.addressof(self.ptrs)
        self.args = (len(states), shape[0] // W, W, slabs, T, n)


def beam_states(states, W) -> BeamStates:
    return BeamStates(states, W)


def beam_reorder(states, parent, length=None, stream=None):
    """Row r of every state becomes what row parent[r] was, in place
    (neon_beam_reorder); length int32 [B W]: the tokens of each row, or None for whole
    rows."""
    device = states.device
    on = _on_current(device, stream)
    N = states.rows
    _check(lib().neon_beam_reorder(
        states.ref, *states.args,
        None if length is None else _i32(length, N, "length", device),
        _i32(parent, N, "parent", device), on))


def pages_workspace(n_pages, B):
    """(workspace bytes, counter bytes) of neon_pages_fork; neon_pages_compact takes
    the workspace alone."""
    L = lib()
    return L.neon_pages_workspace(n_pages, B), L.neon_pages_counters(n_pages)


def _pages(refs, table, kv_len, refs_out, stream):
    """(device, stream, n_pages, rows, max_pages, pointers of refs, table, kv_len and
    refs_out) of a page plan."""
    device = refs.get_device()
    shape = table.shape
    if len(shape) != 2 or kv_len.numel() != shape[0]:
        raise ValueError("table: [B][max_pages], one row per sequence of kv_len")
    n = refs.numel()
    return (device, _on_current(device, stream), n, shape[0], shape[1],
            _i32(refs, n, "refs", device), _i32(table, 1, "table", device),
            _i32(kv_len, 1, "kv_len", device), _i32(refs_out, n, "refs_out", device))


def pages_fork(refs, table, kv_len, page_size, refs_out, table_out, len_out, copies, parent=None,
               keep=None, add=None, stream=None, workspace=None, counters=None):
    """Which pages the sequences hold next (neon_pages_fork): refs int32 [n_pages],
    table int32 [B_in][max_pages], kv_len int32 [B_in]; parent, keep, add int32 [B] or
    None; table_out int32 [B][max_pages], len_out int32 [B], copies (src, dst, rows)
    int32 [B] each.  counters: zero-filled once by the caller (each call leaves it
    zero)."""
    device, on, n, B_in, width, refs, table, kv_len, refs_out = _pages(refs, table, kv_len, refs_out, stream)
    shape = table_out.shape
    if len(shape) != 2 or shape[1] != width:
        raise ValueError("table_out: rows of as many entries as table")
    B = shape[0]
    if workspace is None or counters is None:
        wb, cb = pages_workspace(n, B)
        if workspace is None:
            workspace = _scratch(wb, stream)
        if counters is None:
            counters = _scratch(cb, stream, zero=True)
    src, dst, rows = copies
    _check(lib().neon_pages_fork(
        refs, table, kv_len, B_in,
        None if parent is None else _i32(parent, B, "parent", device),
        None if keep is None else _i32(keep, B, "keep", device),
        None if add is None else _i32(add, B, "add", device), refs_out,
        _i32(table_out, B * width, "table_out", device), _i32(len_out, B, "len_out", device),
        _i32(src, B, "copies[0]", device), _i32(dst, B, "copies[1]", device),
        _i32(rows, B, "copies[2]", device), B, n, page_size, width,
        _buffer(workspace, "workspace", device), workspace.nbytes,
        _buffer(counters, "counters", device), counters.nbytes, on))


class PagedLayers:
    """Caches of one shape and format that share a page table (the layers of a model)."""

    def __init__(self, caches):
        self.caches = tuple(caches)  # keeps them alive
        if not self.caches:
            raise ValueError("PagedLayers: at least one cache")
        first = self.caches[0]
        self.device, self.format = first.device, first.format
        if any(c.device != first.device for c in self.caches):
            raise ValueError("PagedLayers: caches on one device")
        self.structs = (PagedKVStruct * len(self.caches))(*(c.struct for c in self.caches))
        self.ref = C.addressof(self.structs)


def paged_layers(caches) -> PagedLayers:
    return PagedLayers(caches)


def pages_copy(layers, src, dst, rows=None, stream=None):
    """Copies pages src[i] -> dst[i], the first rows[i] tokens of each (None: all), in
    every cache of `layers` (PagedLayers or one PagedKV; neon_pages_copy)."""
    if isinstance(layers, PagedKV):
        layers = PagedLayers([layers])
    device = layers.device
    on = _on_current(device, stream)
    n = src.numel()
    _check(lib().neon_pages_copy(
        layers.ref, len(layers.caches), _i32(src, n, "src", device), _i32(dst, n, "dst", device),
        None if rows is None else _i32(rows, n, "rows", device), n, on))


def pages_compact(refs, table, kv_len, page_size, refs_out, table_out, moved_to, copies, stream=None,
                  workspace=None):
    """Moves the used pages of a pool to its lowest ids (neon_pages_compact): moved_to
    int32 [n_pages], copies (src, dst) int32 [n_pages / 2] each, for pages_copy."""
    device, on, n, B, width, refs, table, kv_len, refs_out = _pages(refs, table, kv_len, refs_out, stream)
    if workspace is None:
        workspace = _scratch(pages_workspace(n, B)[0], stream)
    src, dst = copies
    _check(lib().neon_pages_compact(
        refs, table, kv_len, refs_out, _i32(table_out, B * width, "table_out", device),
        _i32(moved_to, n, "moved_to", device), _i32(src, n // 2, "copies[0]", device),
        _i32(dst, n // 2, "copies[1]", device), B, n, page_size, width,
        _buffer(workspace, "workspace", device), workspace.nbytes, on))


PREFILL_BATCHED, PREFILL_STEPWISE, PREFILL_CHUNKED, PREFILL_MX8 = 0, 1, 2, 3
DECODE_EXACT, DECODE_MATRIX, DECODE_MATRIX_MX8 = 0, 1, 2


# ---------------------------------------------------------------------------
# context-level API
# ---------------------------------------------------------------------------
class Engine:
    """One model context on one device (weights, KV cache, captured step)."""

    def __init__(self, cfg: Config | str = "gpt-oss-20b", device: int = 0, **overrides):
        if isinstance(cfg, str):
            cfg = config_preset(cfg, **overrides)
        self.cfg = cfg
        self._ctx = C.c_void_p()
        _check(lib().neon_ctx_create(C.byref(cfg), device, C.byref(self._ctx)))
        self.batch = 0

    def close(self):
        if self._ctx:
            lib().neon_ctx_destroy(self._ctx)
            self._ctx = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def _chk(self, status):
        _check(status, self._ctx)

    def init_random(self, seed: int = 0, stream=None):
        self._chk(lib().neon_init_random(self._ctx, seed, _stream(stream)))

    def load_tensor(self, name: str, data):
        """data: bytes, memoryview or a C-contiguous numpy array (read in place)."""
        import numpy as np
        a = np.frombuffer(data, dtype=np.uint8) if not isinstance(data, np.ndarray) else data
        if not a.flags.c_contiguous:
            raise ValueError(f"load_tensor({name!r}): data must be contiguous")
        self._chk(lib().neon_load_tensor(self._ctx, name.encode(), C.c_void_p(a.ctypes.data),
                                         a.nbytes))

    def load_checkpoint(self, path: str, strict: bool = True) -> int:
        """Loads a local gpt-oss safetensors checkpoint (file or directory)."""
        from .loader import load_checkpoint
        return load_checkpoint(self, path, strict=strict)

    def tensor_ptr(self, name: str):
        p, n = C.c_void_p(), C.c_size_t()
        self._chk(lib().neon_tensor_ptr(self._ctx, name.encode(), C.byref(p), C.byref(n)))
        return p.value, n.value

    def set_decode_mode(self, mode: int):
        """DECODE_EXACT (default: batched steps bit-identical to batch 1) or
        DECODE_MATRIX (steps of 2+ sequences on the matrix cores; equal to
        the exact steps up to the order of fp32 additions)."""
        self._chk(lib().neon_set_decode_mode(self._ctx, mode))

    def set_prefill_mode(self, mode: int):
        """PREFILL_CHUNKED (default: up to 512 prompt rows per pass), PREFILL_STEPWISE
        (every prompt token as a decode step) or PREFILL_BATCHED (all prompt rows at
        once on the matrix cores; equal to the others up to bf16 rounding)."""
        self._chk(lib().neon_set_prefill_mode(self._ctx, mode))

    def set_sampling(self, temperature: float = 0.0, top_p: float = 1.0, seed: int = 0):
        """temperature 0: greedy; else softmax(logits / temperature) within the
        top-p nucleus, reproducible for a given seed."""
        self._chk(lib().neon_set_sampling(self._ctx, temperature, top_p, seed))

    def prefill(self, ids, stream=None):
        """ids: nested list / array [batch][n_tokens] of int, or a list of
        prompts of different lengths (neon_prefill_ragged)."""
        import numpy as np
        if isinstance(ids, (list, tuple)) and ids and not np.isscalar(ids[0]) and \
                len({len(p) for p in ids}) > 1:
            return self.prefill_ragged(ids, stream)
        a = np.ascontiguousarray(ids, dtype=np.int32)
        if a.ndim == 1:
            a = a[None, :]
        self._chk(lib().neon_prefill(self._ctx, a.ctypes.data_as(C.c_void_p), a.shape[0],
                                     a.shape[1], _stream(stream)))
        self.batch = a.shape[0]

    def prefill_ragged(self, prompts, stream=None):
        """prompts: one sequence of int ids per sequence, lengths free."""
        import numpy as np
        lens = np.ascontiguousarray([len(p) for p in prompts], dtype=np.int32)
        flat = np.ascontiguousarray(np.concatenate([np.asarray(p, np.int64) for p in prompts])
                                    if len(prompts) else np.zeros(0), dtype=np.int32)
        self._chk(lib().neon_prefill_ragged(self._ctx, flat.ctypes.data_as(C.c_void_p),
                                            lens.ctypes.data_as(C.c_void_p), len(prompts),
                                            _stream(stream)))
        self.batch = len(prompts)

    def seq_add(self, prompt, stream=None) -> int:
        """A sequence joins the running batch (neon_seq_add): returns its row."""
        import numpy as np
        ids = np.ascontiguousarray(prompt, dtype=np.int32)
        slot = C.c_int(-1)
        self._chk(lib().neon_seq_add(self._ctx, ids.ctypes.data_as(C.c_void_p), len(ids),
                                     C.byref(slot), _stream(stream)))
        self.batch = max(self.batch, slot.value + 1)
        return slot.value

    def seq_remove(self, slot: int, stream=None):
        """A sequence leaves (neon_seq_remove): its row and KV block are free;
        free rows at the end of the batch leave it."""
        import numpy as np
        held = self.seq_lens() if self.batch else np.zeros(0, np.int32)
        self._chk(lib().neon_seq_remove(self._ctx, slot, _stream(stream)))
        held[slot] = 0
        nz = np.nonzero(held)[0]
        self.batch = int(nz[-1]) + 1 if len(nz) else 0

    def seq_lens(self):
        """Tokens held by each sequence (prompt + generated), int32 [batch]."""
        import numpy as np
        out = np.empty(max(self.batch, 1), np.int32)
        self._chk(lib().neon_seq_lens(self._ctx, out.ctypes.data_as(C.c_void_p)))
        return out[:self.batch]

    def decode(self, n_steps: int, stream=None):
        self._chk(lib().neon_decode(self._ctx, n_steps, _stream(stream)))

    def seq_len(self) -> int:
        n = C.c_int()
        self._chk(lib().neon_seq_len(self._ctx, C.byref(n)))
        return n.value

    def read_tokens(self, start=0, count=None, stream=None):
        import numpy as np
        if count is None:
            count = self.seq_len() - start
        out = np.empty((self.batch, count), np.int32)
        self._chk(lib().neon_read_tokens(self._ctx, start, count,
                                         out.ctypes.data_as(C.c_void_p), _stream(stream)))
        return out

    def read_activation(self, name: str, stream=None):
        """One activation buffer of the last step (see neon_read_activation)."""
        import numpy as np
        c = self.cfg
        if name == "mx_route":
            S = min(c.n_experts, self.batch * c.top_k)
            out = np.empty(66 * S, np.int32)
            self._chk(lib().neon_read_activation(self._ctx, name.encode(),
                                                 out.ctypes.data_as(C.c_void_p), out.nbytes,
                                                 _stream(stream)))
            return out
        if name == "mx_items":  # count, then up to 256 packed work items
            out = np.empty(257, np.int32)
            self._chk(lib().neon_read_activation(self._ctx, name.encode(),
                                                 out.ctypes.data_as(C.c_void_p), out.nbytes,
                                                 _stream(stream)))
            return out
        width = {"hidden": c.hidden, "moe_in": c.hidden, "moe_idx": c.top_k,
                 "moe_score": c.top_k, "qkv": (c.n_heads + 2 * c.n_kv_heads) * c.head_dim,
                 "attn_out": c.n_heads * c.head_dim}[name]
        dt = {"moe_idx": np.int32, "moe_score": np.float32}.get(name, np.uint16)
        out = np.empty((self.batch, width), dt)
        self._chk(lib().neon_read_activation(self._ctx, name.encode(),
                                             out.ctypes.data_as(C.c_void_p), out.nbytes,
                                             _stream(stream)))
        return out

    def read_hidden(self, stream=None):
        return self.read_activation("hidden", stream)

    def read_logits(self, stream=None):
        import numpy as np
        out = np.empty((self.batch, self.cfg.vocab), np.float32)
        self._chk(lib().neon_read_logits(self._ctx, out.ctypes.data_as(C.c_void_p),
                                         _stream(stream)))
        return out
