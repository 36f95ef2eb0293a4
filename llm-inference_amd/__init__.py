"""Python host side of the MI355X (gfx950) decode kernels.

Thin ctypes bindings of libllm_amd.so, whose C ABI (include/llm_amd/kernels.h, forward.h)
replaces the reference's src/kernels.cuh and src/forward.cuh launchers and step API
(William-Lamer/llm-inference). The wrappers take torch tensors for device memory and a torch
stream (or the current one); torch is only the allocator and stream provider. Every call goes to
the HIP kernels: there is no CPU path, and a missing library raises. The launchers are called
through a native module (csrc/launchers.cpp) where one is built for this Python and torch, and
through ctypes otherwise and for arguments that it does not recognise.

Errors the reference reports with exit(EXIT_FAILURE) raise LlmError here (the library is
switched to recording mode on load).
"""
import ctypes
import importlib.machinery
import importlib.util
import os
from pathlib import Path

HERE = Path(__file__).resolve().parent
LIB_PATH = HERE / "libllm_amd.so"
# the module built for this very Python (another's is not looked at)
LAUNCHERS_PATH = HERE / ("_launchers" + importlib.machinery.EXTENSION_SUFFIXES[0])

__all__ = [
    "LlmError", "lib", "embedding_forward", "rmsnorm_forward", "gemv_forward",
    "gemv_residual_forward", "qkv_forward", "gate_up_forward", "qk_norm_rope_forward",
    "qk_norm_rope_rows", "attention_forward", "argmax_forward", "swiglu_forward",
    "attention_workspace_floats", "rmsnorm_qkv_forward", "rmsnorm_gemv_forward",
    "rmsnorm_gate_up_forward", "hbm_stream_probe", "hbm_read_peak_probe", "hbm_copy_peak_probe", "sample_forward",
    "qk_norm_rope_attention_forward", "dump_open",
    "dump_close", "dump_enabled", "attention_forward_noalloc", "EXPORTED_SYMBOLS",
    "qk_norm_rope_attention_one_pass", "attention_one_pass_bytes", "attention_one_pass_supported",
    "ROPE_PLAIN", "ROPE_LINEAR", "ROPE_YARN", "rope_frequencies", "qk_norm_rope_paged",
    "lora_projection_forward", "lora_projection_workspace_floats", "sample_rows_forward",
    "sample_rows_workspace_floats",
    "attention_paged_forward", "attention_paged_workspace_floats", "logits_penalty_forward",
]

# Every symbol include/llm_amd/*.h declares.
EXPORTED_SYMBOLS = [
    "embedding_forward", "rmsnorm_forward", "gemv_forward", "gemv_residual_forward",
    "qkv_forward", "gate_up_forward", "qk_norm_rope_forward", "attention_forward",
    "argmax_forward", "qk_norm_rope_rows", "swiglu_forward", "attention_workspace_floats",
    "rmsnorm_qkv_forward", "rmsnorm_gemv_forward", "rmsnorm_gate_up_forward",
    "hbm_stream_probe", "hbm_read_peak_probe", "hbm_copy_peak_probe", "sample_forward", "sample_temperature",
    "dump_open", "dump_close",
    "dump_enabled", "dump_bf16", "dump_f32", "llm_set_exit_on_error", "llm_last_error", "llm_clear_error",
    "load_config", "load_weights", "free_weights", "print_weight_checksums",
    "alloc_run_state", "free_run_state", "capture_graph", "forward", "sample_argmax",
    "weight_bytes_per_step", "kv_bytes_per_position", "alloc_run_state_seq", "synth_weights",
    "synth_fill", "generate_greedy", "attention_forward_noalloc",
    "qk_norm_rope_attention_forward", "qk_norm_rope_attention_one_pass",
    "attention_one_pass_bytes", "attention_one_pass_supported",
    "rope_frequencies", "qk_norm_rope_paged", "attention_paged_forward",
    "attention_paged_workspace_floats", "logits_penalty_forward", "lora_projection_forward",
    "lora_projection_workspace_floats", "sample_rows_forward", "sample_rows_workspace_floats",
]


class LlmError(RuntimeError):
    """A shape, alignment or HIP error reported by libllm_amd."""


_lib = None
_native = None  # the launchers' module, once the library is loaded; None: every call through ctypes

_vp = ctypes.c_void_p
_i = ctypes.c_int
_f = ctypes.c_float
_sz = ctypes.c_size_t
_i64 = ctypes.c_int64


class PagedBatch(ctypes.Structure):
    """include/llm_amd/paged.h PagedBatch."""
    _fields_ = [("key_cache", _vp), ("value_cache", _vp), ("page_stride", _i64), ("slot_stride", _i64),
                ("head_stride", _i64), ("page_table", _vp), ("q_start", _vp), ("kv_len", _vp),
                ("n_seqs", _i), ("n_pages", _i), ("page_size", _i), ("table_pages", _i),
                ("n_kv_heads", _i), ("head_dim", _i)]


class LoraBatch(ctypes.Structure):
    """include/llm_amd/batch.h LoraBatch."""
    _fields_ = [("a", _vp), ("b", _vp), ("scale", _vp), ("q_start", _vp), ("adapter", _vp),
                ("n_seqs", _i), ("n_adapters", _i), ("rank", _i)]


_SIGS = {
    "embedding_forward": (None, [_vp, _vp, _vp, _i, _vp]),
    "rmsnorm_forward": (None, [_vp, _vp, _vp, _i, _i, _f, _vp]),
    "gemv_forward": (None, [_vp, _vp, _vp, _i, _i, _vp]),
    "gemv_residual_forward": (None, [_vp, _vp, _vp, _i, _i, _vp, _vp]),
    "qkv_forward": (None, [_vp] * 7 + [_i, _i, _i, _vp]),
    "gate_up_forward": (None, [_vp] * 4 + [_i, _i, _vp, _vp, _vp]),
    "qk_norm_rope_forward": (None, [_vp] * 8 + [_i, _i, _i, _f, _f, _vp, _vp, _vp]),
    "qk_norm_rope_rows": (None, [_vp] * 8 + [_i, _i, _i, _i, _f, _f, _vp, _vp, _vp]),
    "attention_forward": (None, [_vp] * 5 + [_i, _i, _i, _vp, _i, _f, _vp]),
    "attention_forward_noalloc": (None, [_vp] * 4 + [_i, _i, _i, _vp, _i, _f, _vp]),
    "argmax_forward": (None, [_vp, _vp, _i, _vp]),
    "swiglu_forward": (None, [_vp, _vp, _vp, _sz, _vp]),
    "attention_workspace_floats": (_sz, [_i, _i, _i]),
    "rmsnorm_qkv_forward": (None, [_vp] * 8 + [_f, _i, _i, _i, _vp]),
    "rmsnorm_gemv_forward": (None, [_vp] * 4 + [_f, _i, _i, _vp]),
    "rmsnorm_gate_up_forward": (None, [_vp] * 5 + [_f, _i, _i, _vp]),
    "hbm_stream_probe": (None, [_vp, _vp, _vp, _sz, _i, _vp]),
    "hbm_read_peak_probe": (None, [_vp, _vp, _sz, _i, _i, _i, _i, _vp]),
    "hbm_copy_peak_probe": (None, [_vp, _vp, _sz, _i, _i, _i, _vp]),
    "qk_norm_rope_attention_forward": (None, [_vp] * 9 + [_vp, _i, _i, _i, _f, _f, _i, _f, _vp]),
    "qk_norm_rope_attention_one_pass": (None, [_vp] * 11 + [_i, _i, _i, _f, _f, _i, _f, _vp]),
    "attention_one_pass_bytes": (_sz, [_i, _i, _i]),
    "attention_one_pass_supported": (_i, [_i, _i, _i, _i]),
    "sample_forward": (None, [_vp, _vp, _i, _f, _f, _vp]),
    "rope_frequencies": (_f, [_vp, _i, ctypes.c_double, _i, ctypes.c_double, _i]),
    "qk_norm_rope_paged": (None, [_vp] * 8 + [_i, _i, _i, _i, _f, _f] + [_i64] * 4 + [_vp]),
    "attention_paged_forward": (None, [_vp] * 4 + [_i] * 5 + [_f, _i64, _i64, _vp]),
    "attention_paged_workspace_floats": (_sz, [_i] * 7),
    "logits_penalty_forward": (None, [_vp] * 12 + [_i] * 5 + [_i64, _i64, _vp]),
    "lora_projection_forward": (None, [_vp] * 6 + [_i] * 3 + [_i64] * 3 + [_vp]),
    "lora_projection_workspace_floats": (_sz, [_i] * 4),
    "sample_rows_forward": (None, [_vp] * 9 + [_i, _i, _i64, _vp]),
    "sample_rows_workspace_floats": (_sz, [_i, _i]),
    "dump_open": (None, [ctypes.c_char_p]),
    "dump_close": (None, []),
    "dump_enabled": (_i, []),
    "dump_bf16": (None, [ctypes.c_char_p, _vp, _i]),
    "dump_f32": (None, [ctypes.c_char_p, _vp, _i]),
    "llm_set_exit_on_error": (_i, [_i]),
    "llm_last_error": (ctypes.c_char_p, []),
    "llm_clear_error": (None, []),
}


def _load_launchers(torch_version):
    """The native launchers, or None where none are built for this Python and torch: their every call
    goes through ctypes as well, with more host time."""
    try:
        name = __name__ + "._launchers"
        loader = importlib.machinery.ExtensionFileLoader(name, str(LAUNCHERS_PATH))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader(name, loader))
        loader.exec_module(module)
    except ImportError:
        return None
    if module.TORCH_VERSION != torch_version.split("+")[0]:
        return None
    module.init(LlmError)
    return module


def lib():
    """The loaded libllm_amd.so (raises LlmError if it has not been built)."""
    global _lib, _native
    if _lib is None:
        # torch first: its bundled HIP runtime then satisfies the library's libamdhip64.so.7
        # dependency (same SONAME), so both share one runtime and torch's streams are valid here.
        import torch
        if not LIB_PATH.exists():
            raise LlmError(f"{LIB_PATH} is missing: build it with `make -C {HERE}` "
                           "(or __graft_entry__.build())")
        L = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in _SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        L.llm_set_exit_on_error(0)
        _lib, _native = L, _load_launchers(torch.__version__)
        from . import model  # noqa: F401  (declares the step API signatures)
        model._declare(L)
    return _lib


def check():
    """Raises LlmError with the library's message if the last call recorded an error."""
    L = lib()
    msg = L.llm_last_error()
    if msg is not None:
        L.llm_clear_error()
        raise LlmError(msg.decode())


def _ptr(t):
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise LlmError("tensors passed to the HIP kernels must live on the GPU")
    if not t.is_contiguous():
        raise LlmError("tensors passed to the HIP kernels must be contiguous")
    return t.data_ptr()


def _bf16(t, name):
    import torch
    if t is not None and not isinstance(t, int) and t.dtype not in (torch.bfloat16, torch.int16,
                                                                     torch.uint16):
        raise LlmError(f"{name} must be bfloat16 (or its raw 16-bit view), got {t.dtype}")
    return _ptr(t)


def _stream(stream):
    import torch
    if stream is None:
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _call(fn, *args):
    fn(*args)
    check()


# ---- launchers (include/llm_amd/kernels.h): the native module first, the general way for what it
# does not recognise ----

def embedding_forward(out, table, d_token, hidden, stream=None):
    if _native and _native.embedding_forward(out, table, d_token, hidden, stream):
        return
    _call(lib().embedding_forward, _bf16(out, "out"), _bf16(table, "table"), _ptr(d_token),
          hidden, _stream(stream))


def rmsnorm_forward(out, inp, weight, rows, dim, eps, stream=None):
    if _native and _native.rmsnorm_forward(out, inp, weight, rows, dim, eps, stream):
        return
    _call(lib().rmsnorm_forward, _bf16(out, "out"), _bf16(inp, "in"), _bf16(weight, "weight"),
          rows, dim, eps, _stream(stream))


def gemv_forward(out, w, x, rows, cols, stream=None):
    if _native and _native.gemv_forward(out, w, x, rows, cols, stream):
        return
    _call(lib().gemv_forward, _bf16(out, "out"), _bf16(w, "w"), _bf16(x, "x"), rows, cols,
          _stream(stream))


def gemv_residual_forward(x, w, inp, rows, cols, tap=None, stream=None):
    if _native and _native.gemv_residual_forward(x, w, inp, rows, cols, tap, stream):
        return
    _call(lib().gemv_residual_forward, _bf16(x, "x"), _bf16(w, "w"), _bf16(inp, "in"), rows,
          cols, _bf16(tap, "tap"), _stream(stream))


def qkv_forward(q, k, v, wq, wk, wv, x, q_rows, kv_rows, cols, stream=None):
    if _native and _native.qkv_forward(q, k, v, wq, wk, wv, x, q_rows, kv_rows, cols, stream):
        return
    _call(lib().qkv_forward, _bf16(q, "q"), _bf16(k, "k"), _bf16(v, "v"), _bf16(wq, "wq"),
          _bf16(wk, "wk"), _bf16(wv, "wv"), _bf16(x, "x"), q_rows, kv_rows, cols,
          _stream(stream))


def gate_up_forward(act, w_gate, w_up, x, rows, cols, gate_tap=None, up_tap=None, stream=None):
    if _native and _native.gate_up_forward(act, w_gate, w_up, x, rows, cols, gate_tap, up_tap,
                                           stream):
        return
    _call(lib().gate_up_forward, _bf16(act, "act"), _bf16(w_gate, "w_gate"), _bf16(w_up, "w_up"),
          _bf16(x, "x"), rows, cols, _bf16(gate_tap, "gate_tap"), _bf16(up_tap, "up_tap"),
          _stream(stream))


def rmsnorm_qkv_forward(q, k, v, wq, wk, wv, x, norm_w, eps, q_rows, kv_rows, cols,
                        stream=None):
    if _native and _native.rmsnorm_qkv_forward(q, k, v, wq, wk, wv, x, norm_w, eps, q_rows, kv_rows,
                                               cols, stream):
        return
    _call(lib().rmsnorm_qkv_forward, _bf16(q, "q"), _bf16(k, "k"), _bf16(v, "v"),
          _bf16(wq, "wq"), _bf16(wk, "wk"), _bf16(wv, "wv"), _bf16(x, "x"),
          _bf16(norm_w, "norm_w"), eps, q_rows, kv_rows, cols, _stream(stream))


def rmsnorm_gemv_forward(out, w, x, norm_w, eps, rows, cols, stream=None):
    if _native and _native.rmsnorm_gemv_forward(out, w, x, norm_w, eps, rows, cols, stream):
        return
    _call(lib().rmsnorm_gemv_forward, _bf16(out, "out"), _bf16(w, "w"), _bf16(x, "x"),
          _bf16(norm_w, "norm_w"), eps, rows, cols, _stream(stream))


def rmsnorm_gate_up_forward(act, w_gate, w_up, x, norm_w, eps, rows, cols, stream=None):
    if _native and _native.rmsnorm_gate_up_forward(act, w_gate, w_up, x, norm_w, eps, rows, cols,
                                                   stream):
        return
    _call(lib().rmsnorm_gate_up_forward, _bf16(act, "act"), _bf16(w_gate, "w_gate"),
          _bf16(w_up, "w_up"), _bf16(x, "x"), _bf16(norm_w, "norm_w"), eps, rows, cols,
          _stream(stream))


def qk_norm_rope_forward(q, k, v, q_norm_w, k_norm_w, key_cache, value_cache, d_pos, n_heads,
                         n_kv_heads, head_dim, eps, theta, q_tap=None, k_tap=None, stream=None):
    if _native and _native.qk_norm_rope_forward(q, k, v, q_norm_w, k_norm_w, key_cache, value_cache,
                                                d_pos, n_heads, n_kv_heads, head_dim, eps, theta,
                                                q_tap, k_tap, stream):
        return
    _call(lib().qk_norm_rope_forward, _bf16(q, "q"), _bf16(k, "k"), _bf16(v, "v"),
          _bf16(q_norm_w, "q_norm_w"), _bf16(k_norm_w, "k_norm_w"), _bf16(key_cache, "key_cache"),
          _bf16(value_cache, "value_cache"), _ptr(d_pos), n_heads, n_kv_heads, head_dim, eps,
          theta, _bf16(q_tap, "q_tap"), _bf16(k_tap, "k_tap"), _stream(stream))


def qk_norm_rope_rows(q, k, v, q_norm_w, k_norm_w, key_cache, value_cache, d_positions,
                      n_tokens, n_heads, n_kv_heads, head_dim, eps, theta, q_tap=None,
                      k_tap=None, stream=None):
    if _native and _native.qk_norm_rope_rows(q, k, v, q_norm_w, k_norm_w, key_cache, value_cache,
                                             d_positions, n_tokens, n_heads, n_kv_heads, head_dim,
                                             eps, theta, q_tap, k_tap, stream):
        return
    _call(lib().qk_norm_rope_rows, _bf16(q, "q"), _bf16(k, "k"), _bf16(v, "v"),
          _bf16(q_norm_w, "q_norm_w"), _bf16(k_norm_w, "k_norm_w"), _bf16(key_cache, "key_cache"),
          _bf16(value_cache, "value_cache"), _ptr(d_positions), n_tokens, n_heads, n_kv_heads,
          head_dim, eps, theta, _bf16(q_tap, "q_tap"), _bf16(k_tap, "k_tap"), _stream(stream))


def attention_workspace_floats(n_heads, head_dim, max_seq):
    return lib().attention_workspace_floats(n_heads, head_dim, max_seq)


def attention_forward(out, q, key_cache, value_cache, att, n_heads, n_kv_heads, head_dim, d_pos,
                      max_seq, scale, stream=None):
    """att: a device pointer (int) to the caller's own allocation of at least [n_heads, max_seq]
    floats (the library checks that allocation's size), or a torch tensor of at least
    attention_workspace_floats(n_heads, head_dim, max_seq) floats: torch's caching allocator
    carves tensors out of larger allocations, whose size says nothing of the tensor's."""
    if _native and _native.attention_forward(out, q, key_cache, value_cache, att, n_heads,
                                             n_kv_heads, head_dim, d_pos, max_seq, scale, stream):
        return
    need = attention_workspace_floats(n_heads, head_dim, max_seq)
    if not isinstance(att, int) and att.numel() < need:
        raise LlmError(f"att holds {att.numel()} floats, attention needs {need}")
    _call(lib().attention_forward, _bf16(out, "out"), _bf16(q, "q"),
          _bf16(key_cache, "key_cache"), _bf16(value_cache, "value_cache"), _ptr(att), n_heads,
          n_kv_heads, head_dim, _ptr(d_pos), max_seq, scale, _stream(stream))


def qk_norm_rope_attention_forward(out, q, k, v, q_norm_w, k_norm_w, key_cache, value_cache, att,
                                   d_pos, n_heads, n_kv_heads, head_dim, eps, theta, max_seq,
                                   scale, stream=None):
    """qk_norm_rope_forward + attention_forward, the QK-norm + RoPE inside the scores pass."""
    if _native and _native.qk_norm_rope_attention_forward(out, q, k, v, q_norm_w, k_norm_w,
                                                          key_cache, value_cache, att, d_pos,
                                                          n_heads, n_kv_heads, head_dim, eps, theta,
                                                          max_seq, scale, stream):
        return
    need = attention_workspace_floats(n_heads, head_dim, max_seq)
    if not isinstance(att, int) and att.numel() < need:
        raise LlmError(f"att holds {att.numel()} floats, attention needs {need}")
    _call(lib().qk_norm_rope_attention_forward, _bf16(out, "out"), _bf16(q, "q"), _bf16(k, "k"),
          _bf16(v, "v"), _bf16(q_norm_w, "q_norm_w"), _bf16(k_norm_w, "k_norm_w"),
          _bf16(key_cache, "key_cache"), _bf16(value_cache, "value_cache"), _ptr(att), _ptr(d_pos),
          n_heads, n_kv_heads, head_dim, eps, theta, max_seq, scale, _stream(stream))


def attention_one_pass_bytes(n_heads, head_dim, max_seq):
    return lib().attention_one_pass_bytes(n_heads, head_dim, max_seq)


def attention_one_pass_supported(n_heads, n_kv_heads, head_dim, max_seq):
    return bool(lib().attention_one_pass_supported(n_heads, n_kv_heads, head_dim, max_seq))


def qk_norm_rope_attention_one_pass(out, q, k, v, q_norm_w, k_norm_w, key_cache, value_cache, ws,
                                    err, d_pos, n_heads, n_kv_heads, head_dim, eps, theta,
                                    max_seq, scale, stream=None):
    """qk_norm_rope_forward + attention_forward in one launch. ws: a zeroed device buffer of
    attention_one_pass_bytes() bytes kept between calls; err: a device int32 (2 on timeout)."""
    need = attention_one_pass_bytes(n_heads, head_dim, max_seq)
    if not isinstance(ws, int) and ws.numel() * ws.element_size() < need:
        raise LlmError(f"ws holds {ws.numel() * ws.element_size()} bytes, one-pass attention "
                       f"needs {need}")
    _call(lib().qk_norm_rope_attention_one_pass, _bf16(out, "out"), _bf16(q, "q"), _bf16(k, "k"),
          _bf16(v, "v"), _bf16(q_norm_w, "q_norm_w"), _bf16(k_norm_w, "k_norm_w"),
          _bf16(key_cache, "key_cache"), _bf16(value_cache, "value_cache"), _ptr(ws), _ptr(err),
          _ptr(d_pos), n_heads, n_kv_heads, head_dim, eps, theta, max_seq, scale,
          _stream(stream))


def attention_forward_noalloc(out, q, key_cache, value_cache, n_heads, n_kv_heads, head_dim,
                              d_pos, max_seq, scale, stream=None):
    """attention_forward with the library's own workspace (allocates nothing)."""
    if _native and _native.attention_forward_noalloc(out, q, key_cache, value_cache, n_heads,
                                                     n_kv_heads, head_dim, d_pos, max_seq, scale,
                                                     stream):
        return
    _call(lib().attention_forward_noalloc, _bf16(out, "out"), _bf16(q, "q"),
          _bf16(key_cache, "key_cache"), _bf16(value_cache, "value_cache"), n_heads, n_kv_heads,
          head_dim, _ptr(d_pos), max_seq, scale, _stream(stream))


def hbm_stream_probe(dst, a, b, n_bytes, mode, stream=None):
    need = (1 << 20) if mode == 0 else n_bytes
    if not isinstance(dst, int) and dst.numel() * dst.element_size() < need:
        raise LlmError(f"dst holds {dst.numel() * dst.element_size()} bytes, the probe needs {need}")
    _call(lib().hbm_stream_probe, _ptr(dst), _ptr(a), _ptr(b), n_bytes, mode, _stream(stream))


def hbm_read_peak_probe(out, a, n_bytes, blocks, threads, loads_in_flight=4, contiguous=0,
                        stream=None):
    """Reads n_bytes of `a` with `blocks` workgroups of `threads` threads, loads_in_flight
    16-byte loads per thread per round, grid-stride (contiguous=0) or one range per workgroup
    (contiguous=1) (the read-peak probe); `out` is a device word written only if a thread's xor
    equals 0x9e3779b9."""
    _call(lib().hbm_read_peak_probe, _ptr(out), _ptr(a), n_bytes, blocks, threads,
          loads_in_flight, contiguous, _stream(stream))


def hbm_copy_peak_probe(dst, a, n_bytes, blocks, threads, chunks_in_flight=4, stream=None):
    """Copies n_bytes of `a` to `dst` grid-stride with `blocks` workgroups of `threads` threads,
    each thread requesting chunks_in_flight 16-byte loads before it stores them (the copy-peak
    probe)."""
    for name, t in (("dst", dst), ("a", a)):
        if not isinstance(t, int) and t.numel() * t.element_size() < n_bytes:
            raise LlmError(f"{name} holds {t.numel() * t.element_size()} bytes, the probe copies "
                           f"{n_bytes}")
    _call(lib().hbm_copy_peak_probe, _ptr(dst), _ptr(a), n_bytes, blocks, threads,
          chunks_in_flight, _stream(stream))


def sample_forward(out, x, n, inv_temp, u, stream=None):
    if _native and _native.sample_forward(out, x, n, inv_temp, u, stream):
        return
    _call(lib().sample_forward, _ptr(out), _bf16(x, "x"), n, inv_temp, u, _stream(stream))


def dump_open(directory):
    """Activation dumps of the eager step into `directory` (include/llm_amd/dump.h)."""
    _call(lib().dump_open, str(directory).encode())


def dump_close():
    lib().dump_close()


def argmax_forward(out, x, n, stream=None):
    if _native and _native.argmax_forward(out, x, n, stream):
        return
    _call(lib().argmax_forward, _ptr(out), _bf16(x, "x"), n, _stream(stream))


def swiglu_forward(act, gate, up, n, stream=None):
    if _native and _native.swiglu_forward(act, gate, up, n, stream):
        return
    _call(lib().swiglu_forward, _bf16(act, "act"), _bf16(gate, "gate"), _bf16(up, "up"), n,
          _stream(stream))


# ---- serving operators over a paged KV cache (include/llm_amd/paged.h). They take tensors alone and
# read every size and stride from them. With a `stream` other than the current one the caller keeps the
# tensors, as they are, until the work on it is done: torch hands a dropped tensor's memory out again ----

ROPE_PLAIN, ROPE_LINEAR, ROPE_YARN = 0, 1, 2


def rope_frequencies(rotary_dim, theta, kind=ROPE_PLAIN, factor=1.0, trained=0):
    """(inv_freq, rope_scale): radians per position of the rotary_dim / 2 rotated pairs, a float64 CPU
    tensor, and the factor of cos and sin, for positions stretched by `kind`."""
    import torch
    inv_freq = torch.zeros(max(rotary_dim // 2, 0), dtype=torch.float64)
    scale = lib().rope_frequencies(inv_freq.data_ptr() or None, rotary_dim, theta, kind, factor, trained)
    check()
    return inv_freq, scale


def _on_device(name, t, dtypes):
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise LlmError(f"{name} must be a tensor on the GPU")
    if t.device.index != torch.cuda.current_device():
        raise LlmError(f"{name} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    if t.dtype not in dtypes:
        raise LlmError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")


def _dense(name, t, dtype, shape):
    """Address of a contiguous tensor of this type and shape; None stays None."""
    if t is None:
        return None
    _on_device(name, t, (dtype,))
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise LlmError(f"{name} must be contiguous of shape {tuple(shape)}, got {tuple(t.shape)}")
    return t.data_ptr()


def _bits16():
    import torch
    return torch.bfloat16, torch.int16, torch.uint16


def _head_rows(name, t, shape):
    """(address, elements between rows) of rows of whole heads, contiguous within a row."""
    _on_device(name, t, _bits16())
    if tuple(t.shape) != tuple(shape):
        raise LlmError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    n, heads, dim = t.shape
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != dim):
        raise LlmError(f"the rows of {name} must be contiguous")
    return t.data_ptr(), t.stride(0) if n > 1 else heads * dim


def _paged_batch(key_cache, value_cache, page_table, q_start, kv_len):
    import torch
    for name, t in (("key_cache", key_cache), ("value_cache", value_cache)):
        _on_device(name, t, _bits16())
        if t.dim() != 4 or t.stride(3) != 1:
            raise LlmError(f"{name} must have shape [pages, slots, kv heads, head_dim], the last contiguous")
    if key_cache.shape != value_cache.shape or key_cache.stride() != value_cache.stride():
        raise LlmError("key_cache and value_cache must have the same shape and strides")
    _on_device("page_table", page_table, (torch.int32,))
    if page_table.dim() != 2:
        raise LlmError(f"page_table must have shape [sequences, pages], got {tuple(page_table.shape)}")
    pages, slots, kv_heads, dim = key_cache.shape
    seqs = page_table.shape[0]
    strides = [s if n > 1 else 0 for n, s in zip(key_cache.shape, key_cache.stride())]
    return PagedBatch(key_cache.data_ptr(), value_cache.data_ptr(), *strides[:3],
                      _dense("page_table", page_table, torch.int32, page_table.shape),
                      _dense("q_start", q_start, torch.int32, (seqs + 1,)),
                      _dense("kv_len", kv_len, torch.int32, (seqs,)),
                      seqs, pages, slots, page_table.shape[1], kv_heads, dim)


def qk_norm_rope_paged(q_out, q, k, v, q_norm_w, k_norm_w, inv_freq, key_cache, value_cache, page_table,
                       q_start, kv_len, eps, rope_scale=1.0, interleaved=False, stream=None):
    """Norm and rotation of q [tokens, heads, head_dim] into q_out and of k into key_cache, v into
    value_cache [pages, slots, kv heads, head_dim], at the places that page_table [sequences, pages], q_start
    [sequences + 1] and kv_len [sequences] give. inv_freq: float64 [rotary_dim / 2] on the GPU. Norm weights
    None: no norm. Rows of q, k, v and q_out may lie apart (slices of one projection's rows)."""
    if _native and _native.qk_norm_rope_paged(q_out, q, k, v, q_norm_w, k_norm_w, inv_freq, key_cache, value_cache,
                                              page_table, q_start, kv_len, eps, rope_scale, interleaved, stream):
        return
    import torch
    batch = _paged_batch(key_cache, value_cache, page_table, q_start, kv_len)
    _on_device("q", q, _bits16())
    if q.dim() != 3:
        raise LlmError(f"q must have shape [tokens, heads, head_dim], got {tuple(q.shape)}")
    n, heads, dim = q.shape[0], q.shape[1], batch.head_dim
    rows = [_head_rows("q_out", q_out, (n, heads, dim)), _head_rows("q", q, (n, heads, dim)),
            _head_rows("k", k, (n, batch.n_kv_heads, dim)), _head_rows("v", v, (n, batch.n_kv_heads, dim))]
    for name, w in (("q_norm_w", q_norm_w), ("k_norm_w", k_norm_w)):
        if w is not None:
            _on_device(name, w, _bits16())
            _dense(name, w, w.dtype, (dim,))
    _on_device("inv_freq", inv_freq, (torch.float64,))
    _dense("inv_freq", inv_freq, torch.float64, (inv_freq.numel(),))
    _call(lib().qk_norm_rope_paged, *(r[0] for r in rows), _ptr(q_norm_w), _ptr(k_norm_w), _ptr(inv_freq),
          ctypes.byref(batch), n, heads, 2 * inv_freq.numel(), int(interleaved), eps, rope_scale,
          *(r[1] for r in rows), _stream(stream))


def attention_paged_workspace_floats(n_tokens, n_seqs, n_heads, n_kv_heads, head_dim, max_q_len, max_kv_len):
    """Floats of ws for attention_paged_forward with these sizes and with any smaller ones of these heads."""
    floats = lib().attention_paged_workspace_floats(n_tokens, n_seqs, n_heads, n_kv_heads, head_dim,
                                                    max_q_len, max_kv_len)
    check()
    return floats


def attention_paged_forward(out, q, key_cache, value_cache, page_table, q_start, kv_len, ws, scale,
                            max_q_len, max_kv_len, window=0, stream=None):
    """Attention of q [tokens, heads, head_dim] over the pages of its rows' sequences, into out. ws: a
    float32 tensor of at least attention_paged_workspace_floats(...) floats for these sizes (None where that
    is 0), kept between calls that do not overlap."""
    if _native and _native.attention_paged_forward(out, q, key_cache, value_cache, page_table, q_start, kv_len, ws,
                                                   scale, max_q_len, max_kv_len, window, stream):
        return
    import torch
    batch = _paged_batch(key_cache, value_cache, page_table, q_start, kv_len)
    _on_device("q", q, _bits16())
    if q.dim() != 3:
        raise LlmError(f"q must have shape [tokens, heads, head_dim], got {tuple(q.shape)}")
    n, heads, dim = q.shape[0], q.shape[1], batch.head_dim
    out_at, out_stride = _head_rows("out", out, (n, heads, dim))
    q_at, q_stride = _head_rows("q", q, (n, heads, dim))
    if ws is not None:
        _on_device("ws", ws, (torch.float32,))
        _dense("ws", ws, torch.float32, ws.shape)
    if n and heads % max(batch.n_kv_heads, 1) == 0:
        need = attention_paged_workspace_floats(n, batch.n_seqs, heads, batch.n_kv_heads, dim, max_q_len,
                                                max_kv_len)
        have = 0 if ws is None else ws.numel()
        if have < need:
            raise LlmError(f"ws holds {have} floats, attention needs {need}")
    _call(lib().attention_paged_forward, out_at, q_at, ctypes.byref(batch), _ptr(ws), n, heads, max_q_len,
          max_kv_len, window, scale, out_stride, q_stride, _stream(stream))


def logits_penalty_forward(out, logits, tokens=None, prompt_len=None, token_len=None, repetition=None,
                           frequency=None, presence=None, bias_tokens=None, bias=None, bias_len=None,
                           allowed=None, stream=None):
    """Penalties over each row's tokens [rows, capacity], biases [rows, capacity] and the mask of allowed
    tokens [rows, words] (int32 words, bit t % 32 of word t / 32) on logits [rows, vocab], into out (which
    may be logits)."""
    if _native and _native.logits_penalty_forward(out, logits, tokens, prompt_len, token_len, repetition, frequency,
                                                  presence, bias_tokens, bias, bias_len, allowed, stream):
        return
    import torch
    for name, t in (("out", out), ("logits", logits)):
        _on_device(name, t, _bits16())
    for name, t in (("out", out), ("logits", logits)):
        if t.dim() != 2 or t.shape != logits.shape or (t.shape[1] > 1 and t.stride(1) != 1):
            raise LlmError(f"{name} must have shape [rows, vocab], the same for both, with contiguous rows")
    rows, vocab = logits.shape
    strides = [t.stride(0) if rows > 1 else max(vocab, 1) for t in (out, logits)]
    wide = {}
    for name, t in (("allowed", allowed), ("tokens", tokens), ("bias_tokens", bias_tokens)):
        if t is not None:
            _on_device(name, t, (torch.int32, torch.uint32) if name == "allowed" else (torch.int32,))
        if t is not None and t.dim() != 2:
            raise LlmError(f"{name} must have two dimensions, got {tuple(t.shape)}")
        wide[name] = 0 if t is None else t.shape[1]
    _call(lib().logits_penalty_forward, out.data_ptr() or None, logits.data_ptr() or None,
          _dense("tokens", tokens, torch.int32, (rows, wide["tokens"])),
          _dense("prompt_len", prompt_len, torch.int32, (rows,)),
          _dense("token_len", token_len, torch.int32, (rows,)),
          _dense("repetition", repetition, torch.float32, (rows,)),
          _dense("frequency", frequency, torch.float32, (rows,)),
          _dense("presence", presence, torch.float32, (rows,)),
          _dense("bias_tokens", bias_tokens, torch.int32, (rows, wide["bias_tokens"])),
          _dense("bias", bias, torch.float32, (rows, wide["bias_tokens"])),
          _dense("bias_len", bias_len, torch.int32, (rows,)),
          allowed if allowed is None else _dense("allowed", allowed, allowed.dtype, (rows, wide["allowed"])),
          rows, vocab, wide["tokens"], wide["bias_tokens"], wide["allowed"], *strides, _stream(stream))


# ---- what the requests of a batch bring of their own (include/llm_amd/batch.h); tensors alone, as above ----

def lora_projection_workspace_floats(n_tokens, n_out, n_in, rank):
    """Floats of ws for lora_projection_forward with these sizes and with fewer tokens or a lower rank (0: no
    adapters)."""
    floats = lib().lora_projection_workspace_floats(n_tokens, n_out, n_in, rank)
    check()
    return floats


def _matrix_rows(name, t, shape):
    """(address, elements between rows) of rows of 16-bit elements, contiguous within a row."""
    _on_device(name, t, _bits16())
    if tuple(t.shape) != tuple(shape) or (shape[1] > 1 and t.stride(1) != 1):
        raise LlmError(f"{name} must have shape {tuple(shape)} with contiguous rows, got {tuple(t.shape)}")
    return t.data_ptr() or None, t.stride(0) if shape[0] > 1 else max(shape[1], 1)


def _workspace(ws, need, what):
    import torch
    if ws is not None:
        _on_device("ws", ws, (torch.float32,))
        _dense("ws", ws, torch.float32, ws.shape)
    have = 0 if ws is None else ws.numel()
    if have < need:
        raise LlmError(f"ws holds {have} floats, {what} needs {need}")
    return _ptr(ws)


def lora_projection_forward(out, x, w=None, lora_a=None, lora_b=None, lora_scale=None, q_start=None, adapter=None,
                            residual=None, ws=None, stream=None):
    """out [tokens, n_out] = residual + x [tokens, n_in] wT, and for the rows q_start[s] .. q_start[s + 1] - 1 of
    sequence s with the adapter a = adapter[s] + lora_scale[a] (x lora_a[a]T) lora_b[a]T. w [n_out, n_in], lora_a
    [adapters, rank, n_in], lora_b [adapters, n_out, rank]; each of w, the adapters (lora_a, lora_b, q_start and
    adapter together), lora_scale and residual may be None. ws: a float32 tensor of at least
    lora_projection_workspace_floats(...) floats (None where that is 0), kept between calls that do not overlap."""
    if _native and _native.lora_projection_forward(out, x, w, lora_a, lora_b, lora_scale, q_start, adapter, residual,
                                                   ws, stream):
        return
    import torch
    for name, t in (("out", out), ("x", x)):
        _on_device(name, t, _bits16())
        if t.dim() != 2:
            raise LlmError(f"{name} must have two dimensions, got {tuple(t.shape)}")
    n, n_in, n_out = x.shape[0], x.shape[1], out.shape[1]
    out_at, out_stride = _matrix_rows("out", out, (n, n_out))
    x_at, x_stride = _matrix_rows("x", x, (n, n_in))
    residual_at, residual_stride = (None, n_out) if residual is None else _matrix_rows("residual", residual, (n, n_out))
    if w is not None:
        _on_device("w", w, _bits16())
        _dense("w", w, w.dtype, (n_out, n_in))
    batch, rank = None, 0
    parts = dict(lora_a=lora_a, lora_b=lora_b, q_start=q_start, adapter=adapter)
    if any(t is not None for t in parts.values()) or lora_scale is not None:
        for name, t in parts.items():
            if t is None:
                raise LlmError(f"adapters need lora_a, lora_b, q_start and adapter: {name} is None")
        for name, t in (("lora_a", lora_a), ("lora_b", lora_b)):
            _on_device(name, t, _bits16())
        if lora_a.dim() != 3:
            raise LlmError(f"lora_a must have shape [adapters, rank, n_in], got {tuple(lora_a.shape)}")
        _on_device("adapter", adapter, (torch.int32,))
        adapters, rank, seqs = lora_a.shape[0], lora_a.shape[1], adapter.numel()
        batch = LoraBatch(_dense("lora_a", lora_a, lora_a.dtype, (adapters, rank, n_in)),
                          _dense("lora_b", lora_b, lora_b.dtype, (adapters, n_out, rank)),
                          _dense("lora_scale", lora_scale, torch.float32, (adapters,)),
                          _dense("q_start", q_start, torch.int32, (seqs + 1,)),
                          _dense("adapter", adapter, torch.int32, (seqs,)), seqs, adapters, rank)
    ws_at = _workspace(ws, lora_projection_workspace_floats(n, n_out, n_in, rank), "the projection")
    _call(lib().lora_projection_forward, out_at, x_at, _ptr(w), residual_at,
          None if batch is None else ctypes.byref(batch), ws_at, n, n_out, n_in, out_stride, x_stride,
          residual_stride, _stream(stream))


def sample_rows_workspace_floats(rows, vocab):
    """Floats of ws for sample_rows_forward with these sizes and with smaller ones."""
    floats = lib().sample_rows_workspace_floats(rows, vocab)
    check()
    return floats


def sample_rows_forward(out, logits, u, temperature=None, top_k=None, top_p=None, min_p=None, logprob=None, ws=None,
                        stream=None):
    """A token of each row of logits [rows, vocab] into out (int32 [rows]), drawn with the given u (float32 [rows],
    in [0, 1)) from what temperature, top_k, top_p and min_p ([rows] each, or None: off) leave; logprob (float32
    [rows]): ln of its probability there. ws: a float32 tensor of at least sample_rows_workspace_floats(...) floats
    (None where that is 0), kept between calls that do not overlap."""
    if _native and _native.sample_rows_forward(out, logits, u, temperature, top_k, top_p, min_p, logprob, ws, stream):
        return
    import torch
    _on_device("logits", logits, _bits16())
    if logits.dim() != 2:
        raise LlmError(f"logits must have shape [rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    logits_at, stride = _matrix_rows("logits", logits, (rows, vocab))
    f32, i32 = torch.float32, torch.int32
    columns = [_dense(name, t, dtype, (rows,)) for name, t, dtype in (
        ("out", out, i32), ("logprob", logprob, f32), ("temperature", temperature, f32), ("top_k", top_k, i32),
        ("top_p", top_p, f32), ("min_p", min_p, f32), ("u", u, f32))]
    ws_at = _workspace(ws, sample_rows_workspace_floats(rows, vocab), "the draw")
    _call(lib().sample_rows_forward, columns[0], columns[1], logits_at, *columns[2:], ws_at, rows, vocab, stride,
          _stream(stream))
