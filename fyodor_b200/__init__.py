"""fyodor_b200 - Python mirror of the Fyodor provider interface for B200.

The product is the C-ABI library ``libfyodor_b200.so`` next to this file
(built by ``fyodor_b200.build``). This module binds it with ctypes and
exposes the same operations the engine reaches through its compute layer
(backend/include/compute.h): typed matvec/matmul on a provider context,
resident plans (create, token, prefill, stats, KV snapshot), plus the
device-level extensions declared in include/fyodor_b200.h.

There is no CPU fallback: if the library is missing, importing the module
raises; if the provider declines (no B200), ``Provider()`` raises.
"""
import ctypes as C
import os

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("FYB_LIBRARY") or os.path.join(HERE, "libfyodor_b200.so")  # override: another build

# GGML storage ids (backend/core/llm_internal.h:11-19)
F32, F16, Q4_0, Q8_0, Q4_K, Q6_K, BF16 = 0, 1, 2, 8, 12, 14, 30
BLOCK = {F32: (1, 4), F16: (1, 2), BF16: (1, 2), Q4_0: (32, 18), Q8_0: (32, 34), Q4_K: (256, 144), Q6_K: (256, 210)}


def row_bytes(type_id, cols):
    vals, nbytes = BLOCK[type_id]
    return cols // vals * nbytes


class ComputeStats(C.Structure):
    """nya_compute_stats (backend/include/compute.h:13-22)."""
    _fields_ = [("weights_bytes", C.c_size_t), ("kv_bytes", C.c_size_t), ("scratch_bytes", C.c_size_t),
                ("prefill_batch", C.c_size_t), ("external_matmul_bytes", C.c_size_t),
                ("kernel_launches", C.c_ulonglong), ("uploads", C.c_ulonglong), ("downloads", C.c_ulonglong),
                ("synchronizations", C.c_ulonglong), ("external_matmul_calls", C.c_ulonglong),
                ("graph_captures", C.c_ulonglong), ("graph_replays", C.c_ulonglong),
                ("external_matmul_kind", C.c_uint), ("cutlass_matmul_calls", C.c_ulonglong),
                ("tiled_attention_calls", C.c_ulonglong)]

    def as_dict(self):
        return {k: getattr(self, k) for k, _ in self._fields_}


_P = C.c_void_p
_CREATE = C.CFUNCTYPE(_P)
_DESTROY = C.CFUNCTYPE(None, _P)
_ACTIVE = C.CFUNCTYPE(C.c_int, _P)
_MATVEC = C.CFUNCTYPE(C.c_int, _P, _P, C.c_size_t, C.c_size_t, C.c_uint, _P, _P)
_PLAN_CREATE = C.CFUNCTYPE(_P, _P, _P, C.c_size_t)
_PLAN_FREE = C.CFUNCTYPE(None, _P)
_PLAN_TOKEN = C.CFUNCTYPE(C.c_int, _P, C.c_uint32, C.c_size_t, C.c_int, _P)
_PLAN_PREFILL = C.CFUNCTYPE(C.c_int, _P, _P, C.c_size_t, C.c_size_t, _P)
_PLAN_STATS = C.CFUNCTYPE(None, _P, C.POINTER(ComputeStats))
_MATMUL = C.CFUNCTYPE(C.c_int, _P, _P, C.c_size_t, C.c_size_t, C.c_uint, _P, _P, C.c_size_t)
_ATTN = C.CFUNCTYPE(C.c_int, _P, _P)
_READ_KV = C.CFUNCTYPE(C.c_int, _P, C.c_size_t, C.c_size_t, C.c_size_t, _P, _P, C.c_size_t)


class BackendInterface(C.Structure):
    """nya_backend_interface (backend/include/compute_backend.h:12-29)."""
    _fields_ = [("type", C.c_int), ("name", C.c_char_p), ("capabilities", C.c_uint),
                ("create", _CREATE), ("destroy", _DESTROY), ("active", _ACTIVE), ("matvec", _MATVEC),
                ("plan_create", _PLAN_CREATE), ("plan_free", _PLAN_FREE), ("plan_token", _PLAN_TOKEN),
                ("plan_prefill", _PLAN_PREFILL), ("plan_stats", _PLAN_STATS), ("matmul", _MATMUL),
                ("attention_f32", _P), ("plan_read_kv", _READ_KV), ("context_stats", _P)]


class Tensor(C.Structure):
    """nya_llm_tensor (backend/core/llm_internal.h:22-31)."""
    _fields_ = [("name", C.c_char * 128), ("type", C.c_uint32), ("dimension_count", C.c_uint32),
                ("dimensions", C.c_uint64 * 4), ("relative_offset", C.c_uint64), ("data", C.POINTER(C.c_ubyte)),
                ("data_size", C.c_size_t), ("bound", C.c_int)]


class SynthConfig(C.Structure):
    """fyb_synth_config (include/fyodor_b200.h)."""
    _fields_ = [("layers", C.c_uint32), ("embedding", C.c_uint32), ("heads", C.c_uint32),
                ("kv_heads", C.c_uint32), ("feed_forward", C.c_uint32), ("vocabulary", C.c_uint32),
                ("context", C.c_uint32), ("matrix_type", C.c_uint32), ("embed_type", C.c_uint32),
                ("output_type", C.c_uint32), ("rope_base", C.c_float), ("epsilon", C.c_float),
                ("seed", C.c_uint64), ("norm_mode", C.c_int), ("threads", C.c_int), ("centered", C.c_int),
                ("path", C.c_char_p)]


class KV8CacheDesc(C.Structure):
    """fyb_kv8_cache (include/fyodor_b200.h)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("blocks", C.c_uint32), ("kv_heads", C.c_uint32), ("block_size", C.c_uint32),
                ("head_dim", C.c_uint32), ("format", C.c_uint32)]


class KV8Handle(C.Structure):
    """A cache and its GPU, as the calls on torch tensors take it (csrc/tensors.cc)."""
    _fields_ = [("cache", KV8CacheDesc), ("device", C.c_int32)]


class KV4CacheDesc(C.Structure):
    """fyb_kv4_cache (include/fyodor_b200.h)."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("blocks", C.c_uint32), ("kv_heads", C.c_uint32), ("block_size", C.c_uint32),
                ("head_dim", C.c_uint32)]


class KV4Handle(C.Structure):
    """The same as KV8Handle for a 4-bit cache."""
    _fields_ = [("cache", KV4CacheDesc), ("device", C.c_int32)]


class RopeDesc(C.Structure):
    """fyb_rope_desc (include/fyodor_b200.h)."""
    _fields_ = [("cos_table", C.c_void_p), ("sin_table", C.c_void_p), ("table_rows", C.c_uint32),
                ("dims", C.c_uint32), ("layout", C.c_uint32)]


class RopeScaling(C.Structure):
    """fyb_rope_scaling (include/fyodor_b200.h)."""
    _fields_ = [("kind", C.c_uint32), ("factor", C.c_float), ("original_context", C.c_float),
                ("beta_fast", C.c_float), ("beta_slow", C.c_float), ("low_freq", C.c_float),
                ("high_freq", C.c_float)]


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError("libfyodor_b200.so is not built; run `python -m fyodor_b200.build`")
    lib = C.CDLL(LIB_PATH)
    lib.nya_cuda_backend.restype = C.POINTER(BackendInterface)
    lib.fyb_version.restype = C.c_char_p
    lib.fyb_device_count.restype = C.c_int
    lib.fyb_dequantize.argtypes = [_P, C.c_size_t, C.c_uint, _P, _P]
    lib.fyb_quant_matmul_workspace.restype = C.c_size_t
    lib.fyb_quant_matmul_workspace.argtypes = [C.c_size_t, C.c_size_t, C.c_uint, C.c_size_t]
    lib.fyb_quant_matmul.argtypes = [_P, C.c_size_t, C.c_size_t, C.c_uint, _P, _P, C.c_size_t, _P, C.c_size_t, _P]
    lib.fyb_quant_repack.argtypes = [_P, C.c_size_t, C.c_size_t, C.c_uint, _P, C.c_size_t, _P]
    lib.fyb_quant_matmul_prepared.argtypes = [C.c_size_t, C.c_size_t, C.c_uint, _P, _P, C.c_size_t, _P,
                                              C.c_size_t, _P]
    lib.fyb_attention_workspace.restype = C.c_size_t
    lib.fyb_attention_workspace.argtypes = [C.c_uint] * 5
    lib.fyb_attention_decode.argtypes = [_P, _P, _P, C.c_size_t, _P, C.c_uint, C.c_uint, C.c_uint, C.c_uint,
                                         C.c_uint, C.c_float, _P, C.c_uint, _P, C.c_size_t, _P]
    lib.fyb_attention_verify.argtypes = [_P, _P, _P, C.c_size_t, _P, C.c_uint, C.c_uint, C.c_uint, C.c_uint,
                                         C.c_uint, C.c_uint, C.c_float, _P, C.c_uint, _P, C.c_size_t, _P]
    lib.fyb_attention_decode_static.argtypes = [_P, _P, _P, C.c_size_t, _P, C.c_uint, C.c_uint, C.c_uint, C.c_uint,
                                                C.c_uint, C.c_float, _P, C.c_uint, _P]
    u32, size = C.c_uint32, C.c_size_t
    lib.fyb_kv_blocks.argtypes = [_P, _P, u32, _P, size, u32, _P, _P, _P, _P, _P, _P, _P, _P, u32, _P, _P]
    lib.fyb_kv_release.argtypes = [_P, _P, u32, _P, size, u32, _P, _P, u32, _P]
    lib.fyb_rope_frequencies.argtypes = [u32, C.c_float, C.POINTER(RopeScaling), _P, _P, _P]
    lib.fyb_rope_tables.argtypes = [_P, u32, C.c_float, u32, u32, _P, _P, _P]
    lib.fyb_rope.argtypes = [C.POINTER(RopeDesc), _P, size, u32, u32, _P, size, _P, size, u32, _P, size, _P, size, u32,
                             _P, _P]
    lib.fyb_kv8_append.argtypes = [C.POINTER(KV8CacheDesc), _P, size, u32, _P, size, _P, size, C.POINTER(RopeDesc), _P,
                                   _P, size, _P, size, u32, _P, _P]
    lib.fyb_kv8_read.argtypes = [C.POINTER(KV8CacheDesc), _P, size, _P, _P, _P, _P]
    lib.fyb_kv8_attention_workspace.restype = size
    lib.fyb_kv8_attention_workspace.argtypes = [u32] * 5
    lib.fyb_kv8_attention.argtypes = [C.POINTER(KV8CacheDesc), _P, _P, u32, u32, size, _P, size, u32, _P, size, _P,
                                      size, u32, C.c_float, _P, size, _P, _P]
    for name in ("append", "read", "attention_workspace", "attention"):  # the same but for the cache
        f, g = getattr(lib, "fyb_kv4_" + name), getattr(lib, "fyb_kv8_" + name)
        f.restype = g.restype
        f.argtypes = [C.POINTER(KV4CacheDesc) if a is C.POINTER(KV8CacheDesc) else a for a in g.argtypes]
    lib.fyb_logprobs_workspace.restype = size
    lib.fyb_logprobs_workspace.argtypes = [size, u32, u32]
    lib.fyb_logprobs.argtypes = [u32, _P, size, size, u32, _P, _P, _P, _P, u32, _P, _P, _P, size, _P, _P]
    lib.fyb_plan_tp_info.argtypes = [_P, _P, _P]
    lib.fyb_plan_tp_handle.argtypes = [_P, _P, C.c_size_t]
    lib.fyb_plan_tp_connect.argtypes = [_P, _P, C.c_size_t]
    lib.fyb_plan_tp_disconnect.argtypes = [_P]
    lib.fyb_plan_tp_connect_local.argtypes = [_P, C.POINTER(C.c_void_p), C.c_size_t]
    lib.fyb_plan_error.argtypes = [_P]
    lib.fyb_plan_trace.restype = C.c_long
    lib.fyb_plan_trace.argtypes = [_P, C.c_uint32, C.c_size_t, _P, C.c_size_t, _P, _P, C.c_size_t]
    lib.fyb_plan_decode_greedy.argtypes = [_P, C.c_uint32, C.c_size_t, C.c_size_t, _P]
    lib.fyb_plan_verify.argtypes = [_P, _P, C.c_size_t, C.c_size_t, _P]
    lib.fyb_plan_time_greedy.restype = C.c_double
    lib.fyb_plan_time_greedy.argtypes = [_P, C.c_uint32, C.c_size_t, C.c_size_t]
    lib.fyb_plan_launches_per_token.restype = C.c_ulonglong
    lib.fyb_plan_launches_per_token.argtypes = [_P]
    lib.fyb_plan_decode_form.restype = C.c_int
    lib.fyb_plan_decode_form.argtypes = [_P]
    lib.fyb_plan_profile.argtypes = [_P, C.c_uint32, C.c_size_t, C.c_size_t, _P]
    lib.fyb_plan_time_projection.restype = C.c_double
    lib.fyb_plan_time_projection.argtypes = [_P, C.c_uint, C.c_uint, C.c_uint, C.POINTER(C.c_size_t)]
    lib.fyb_batch_create.restype = _P
    lib.fyb_batch_create.argtypes = [_P, C.c_uint]
    lib.fyb_batch_create_kv8.restype = _P
    lib.fyb_batch_create_kv8.argtypes = [_P, C.c_uint, C.c_uint32, C.c_uint32, C.c_uint32]
    lib.fyb_batch_create_kv4.restype = _P
    lib.fyb_batch_create_kv4.argtypes = [_P, C.c_uint, C.c_uint32, C.c_uint32]
    lib.fyb_batch_score.argtypes = [_P, _P, _P, _P, _P, _P, _P, C.c_uint32, _P, _P]
    lib.fyb_batch_free_blocks.restype = C.c_long
    lib.fyb_batch_free_blocks.argtypes = [_P]
    lib.fyb_batch_free.argtypes = [_P]
    lib.fyb_batch_step.argtypes = [_P, _P, _P, _P, _P]
    lib.fyb_batch_decode_greedy.argtypes = [_P, _P, _P, C.c_size_t, _P]
    lib.fyb_batch_time_greedy.restype = C.c_double
    lib.fyb_batch_time_greedy.argtypes = [_P, _P, _P, C.c_size_t]
    lib.fyb_batch_launches_per_step.restype = C.c_ulonglong
    lib.fyb_batch_launches_per_step.argtypes = [_P]
    lib.fyb_synth_create.restype = _P
    lib.fyb_synth_create.argtypes = [C.POINTER(SynthConfig)]
    lib.fyb_synth_free.argtypes = [_P]
    lib.fyb_synth_fill.argtypes = [_P, C.c_size_t, C.c_size_t, C.c_uint32, C.c_uint64, C.c_uint64]
    return lib


lib = _load()

# exported names declared in include/fyodor_b200.h
EXPORTS = ["nya_cuda_backend", "fyb_version", "fyb_device_count", "fyb_dequantize", "fyb_quant_matmul_workspace",
           "fyb_quant_matmul", "fyb_quant_repack", "fyb_quant_matmul_prepared", "fyb_attention_workspace",
           "fyb_attention_decode", "fyb_attention_verify",
           "fyb_attention_decode_static", "fyb_kv_blocks", "fyb_kv_release", "fyb_rope_frequencies", "fyb_rope_tables",
           "fyb_rope", "fyb_kv8_append", "fyb_kv8_read", "fyb_kv8_attention_workspace", "fyb_kv8_attention",
           "fyb_kv4_append", "fyb_kv4_read", "fyb_kv4_attention_workspace", "fyb_kv4_attention",
           "fyb_logprobs_workspace", "fyb_logprobs",
           "fyb_plan_decode_greedy", "fyb_plan_verify",
           "fyb_plan_time_greedy", "fyb_plan_launches_per_token", "fyb_plan_decode_form", "fyb_plan_profile", "fyb_plan_trace",
           "fyb_plan_tp_info", "fyb_plan_tp_handle", "fyb_plan_tp_connect", "fyb_plan_tp_disconnect",
           "fyb_plan_tp_connect_local", "fyb_plan_error", "fyb_plan_time_projection",
           "fyb_batch_create", "fyb_batch_create_kv8", "fyb_batch_create_kv4", "fyb_batch_score", "fyb_batch_free_blocks", "fyb_batch_free", "fyb_batch_step", "fyb_batch_decode_greedy", "fyb_batch_time_greedy",
           "fyb_batch_launches_per_step",
           "fyb_synth_create",
           "fyb_synth_free", "fyb_synth_fill"]


def _ptr(a):
    return C.c_void_p(a.ctypes.data) if a is not None else None


def api():
    return lib.nya_cuda_backend().contents


# ---------------------------------------------------------------- models
class SynthModel:
    """A seeded random model in the engine's binding layout (fyb_synth_create)."""

    def __init__(self, layers=2, embedding=512, heads=4, kv_heads=2, feed_forward=1024, vocabulary=1024,
                 context=512, matrix_type=Q4_K, embed_type=Q6_K, output_type=Q6_K, rope_base=500000.0,
                 epsilon=1e-5, seed=1234, norm_mode=2, threads=0, centered=0, path=None):
        cfg = SynthConfig(layers, embedding, heads, kv_heads, feed_forward, vocabulary, context, matrix_type,
                          embed_type, output_type, rope_base, epsilon, seed, norm_mode, threads, centered,
                          path.encode() if path else None)
        self.config = cfg
        self.ptr = lib.fyb_synth_create(C.byref(cfg))
        if not self.ptr:
            raise ValueError("invalid synthetic model configuration")
        self.vocabulary = vocabulary
        self.embedding = embedding
        self.layers = layers
        self.kv_dim = embedding // heads * kv_heads
        self.head_dim = embedding // heads
        self.heads, self.kv_heads = heads, kv_heads

    def tensor(self, index):
        """The index-th nya_llm_tensor (0 token_embd, 1 output_norm, 2 output, then 9 per layer)."""
        # nya_llm_context.tensors is at the offset recorded in the ABI golden file (80)
        tensors = C.cast(C.c_void_p.from_address(self.ptr + 80).value, C.POINTER(Tensor))
        return tensors[index]

    def tensor_bytes(self, index):
        t = self.tensor(index)
        return np.ctypeslib.as_array(t.data, shape=(t.data_size,))

    def close(self):
        if self.ptr:
            lib.fyb_synth_free(self.ptr)
            self.ptr = None

    def __del__(self):
        self.close()


# ---------------------------------------------------------------- paged 8-bit and 4-bit KV caches, log probabilities
# The calls below take torch tensors on the current CUDA device and run on
# torch's current stream of it unless `stream` (a cudaStream_t as an int) is
# given. Nothing synchronizes. A refused argument raises ValueError and leaves
# every output as it was.
KV8_INT8, KV8_E4M3 = 0, 1
KV8_FORMATS = {"int8": KV8_INT8, "e4m3": KV8_E4M3}
ROPE_KINDS = {"plain": 0, "linear": 1, "ntk": 2, "yarn": 3, "bands": 4}
_native = None


def _bind_tensors():
    """The extension that takes torch tensors (csrc/tensors.cc), bound to the library on first use."""
    global _native
    if _native is None:
        import torch  # noqa: F401  (the extension links against it)
        from . import _tensors as ext
        ext.bind(*(C.cast(f, C.c_void_p).value for f in (lib.fyb_kv_blocks, lib.fyb_kv_release, lib.fyb_rope,
                                                         lib.fyb_kv8_append, lib.fyb_kv8_read, lib.fyb_kv8_attention,
                                                         lib.fyb_kv4_append, lib.fyb_kv4_read, lib.fyb_kv4_attention,
                                                         lib.fyb_logprobs)))
        _native = ext
    return _native


def _format(name):
    if name not in KV8_FORMATS:
        raise ValueError("the format of an 8-bit cache is one of %s" % sorted(KV8_FORMATS))
    return KV8_FORMATS[name]


def _check(r, what):
    if r == -1:
        raise ValueError("%s refused its arguments" % what)
    if r:
        raise RuntimeError("%s failed to launch (%d)" % (what, r))


def kv_blocks(lengths, new_tokens, table, free_list, free_count, block_size, lengths_out, free_count_out, row_start,
              slots, positions, row_request, status, stream=None):
    """Block tables and slot maps of one serving step (fyb_kv_blocks). All
    int32: lengths, new_tokens, lengths_out and status [requests]; table
    [requests][blocks], extended in place; free_list with free_count [1]
    entries; row_start [requests + 1]; slots, positions and row_request
    [max_rows]."""
    (_native or _bind_tensors()).kv_blocks(lengths, new_tokens, table, free_list, free_count, block_size, lengths_out,
                                      free_count_out, row_start, slots, positions, row_request, status, stream)


def kv_release(lengths, keep, table, free_list, free_count, block_size, stream=None):
    """Shorten every request to keep[r] tokens and give back the blocks it
    needs no more (fyb_kv_release, in place): 0 for a finished request, the
    accepted prefix for one whose draft was rejected."""
    (_native or _bind_tensors()).kv_release(lengths, keep, table, free_list, free_count, block_size, stream)


def rope_frequencies(dims, base, kind="plain", factor=1.0, original_context=0.0, beta_fast=0.0, beta_slow=0.0,
                     low_freq=0.0, high_freq=0.0, factors=None):
    """(frequencies [dims / 2] F32, magnitude) of rotary positions, scaled for
    long contexts by `kind` (fyb_rope_frequencies; host arrays)."""
    if kind not in ROPE_KINDS:
        raise ValueError("kind is one of %s" % sorted(ROPE_KINDS))
    sc = RopeScaling(ROPE_KINDS[kind], factor, original_context, beta_fast, beta_slow, low_freq, high_freq)
    freq, mag = np.empty(max(0, dims) // 2, np.float32), C.c_float(0)
    if factors is not None:
        factors = np.ascontiguousarray(factors, np.float32)
        if factors.size != freq.size:
            raise ValueError("factors has %d entries, %d are needed" % (factors.size, freq.size))
    _check(lib.fyb_rope_frequencies(max(0, dims), base, C.byref(sc), _ptr(factors), _ptr(freq), C.byref(mag)),
           "fyb_rope_frequencies")
    return freq, mag.value


def rope_tables(freq, magnitude, rows, first=0, stream=None):
    """cos and sin [rows][len(freq)] of positions first .. first + rows (device tensors; freq on the device)."""
    import torch
    if not freq.is_cuda or freq.dtype != torch.float32 or not freq.is_contiguous() or \
            freq.get_device() != torch.cuda.current_device():
        raise ValueError("freq has to be a contiguous float32 tensor on the current CUDA device")
    c, s = (torch.empty((rows, freq.numel()), dtype=torch.float32, device=freq.device) for _ in range(2))
    if stream is None:
        stream = torch.cuda.current_stream(freq.device).cuda_stream
    _check(lib.fyb_rope_tables(freq.data_ptr(), 2 * freq.numel(), magnitude, first, rows, c.data_ptr(), s.data_ptr(),
                               stream), "fyb_rope_tables")
    return c, s


def rope(q, k, positions, cos, sin, layout, q_out, k_out, error=None, stream=None):
    """q_out, k_out = q, k [rows][heads][head_dim] rotated to positions[row]
    by the tables (fyb_rope); k and k_out may be None; outputs may be their inputs."""
    (_native or _bind_tensors()).rope(q, k, positions, cos, sin, layout, q_out, k_out, error, stream)


class KV8Cache:
    """A paged 8-bit KV cache over tensors of the caller: k and v
    [blocks][kv_heads][block_size][head_dim] int8 or float8_e4m3fn, k_scale
    and v_scale [blocks][kv_heads] float32 (fyb_kv8_cache)."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch
        kinds = {torch.int8: KV8_INT8, torch.float8_e4m3fn: KV8_E4M3}
        if k.dim() != 4 or k.shape != v.shape or k.dtype not in kinds or k_scale.shape != k.shape[:2] or \
                v_scale.shape != k.shape[:2]:
            raise ValueError("k, v: [blocks][kv_heads][block_size][head_dim] int8 or float8_e4m3fn; scales "
                             "[blocks][kv_heads]")
        for name, t, kind in (("k", k, k.dtype), ("v", v, k.dtype), ("k_scale", k_scale, torch.float32),
                              ("v_scale", v_scale, torch.float32)):
            if t.dtype is not kind or not t.is_cuda or not t.is_contiguous() or t.device != k.device:
                raise ValueError("%s has to be a contiguous %s tensor on the cache's GPU" % (name, kind))
        self.tensors = k, v, k_scale, v_scale
        blocks, self.kv_heads, self.block_size, self.head_dim = k.shape
        self._held = KV8Handle(KV8CacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks,
                                            self.kv_heads, self.block_size, self.head_dim, kinds[k.dtype]),
                               k.get_device())
        self.desc, self._handle = self._held.cache, C.addressof(self._held)

    @classmethod
    def empty(cls, blocks, kv_heads, block_size, head_dim, format="int8", device="cuda"):
        """A cache of its own tensors."""
        import torch
        kind = (torch.int8, torch.float8_e4m3fn)[_format(format)]
        k, v = (torch.zeros((blocks, kv_heads, block_size, head_dim), dtype=torch.int8, device=device).view(kind)
                for _ in range(2))
        return cls(k, v, *(torch.zeros((blocks, kv_heads), device=device) for _ in range(2)))

    def append(self, k, v, slots, positions=None, cos=None, sin=None, layout="interleaved", q=None, q_out=None,
               error=None, stream=None):
        """Store K and V rows [rows][kv_heads][head_dim] at slots[row]
        (fyb_kv8_append). With cos / sin K is rotated to positions[row] first,
        and q to q_out in the same call."""
        (_native or _bind_tensors()).append(self._handle, k, v, slots, positions, cos, sin, layout, q, q_out, error, stream)

    def read(self, slots, k_out, v_out, error=None, stream=None):
        """The values held at slots into k_out, v_out [len(slots)][kv_heads][head_dim] float32 (fyb_kv8_read)."""
        (_native or _bind_tensors()).read(self._handle, slots, k_out, v_out, error, stream)

    def attention_workspace(self, requests, most_rows, heads):
        """A zeroed workspace for attention() calls of this size (one for each stream that calls)."""
        import torch
        need = lib.fyb_kv8_attention_workspace(requests, most_rows, heads, self.kv_heads, self.head_dim)
        if not need:
            raise ValueError("no attention of %d requests, %d rows, %d heads over %d KV heads of %d" %
                             (requests, most_rows, heads, self.kv_heads, self.head_dim))
        return torch.zeros(need, dtype=torch.uint8, device=self.tensors[0].device)

    def attention(self, q, lengths, table, out, workspace, row_start=None, most_rows=1, scale=None, error=None,
                  stream=None):
        """out = causal attention of each request's newest rows over its
        blocks (fyb_kv8_attention): q, out [rows][heads][head_dim], lengths
        [requests], table [requests][blocks]; row_start [requests + 1] where a
        request has other than one row, at most most_rows each."""
        (_native or _bind_tensors()).attention(self._handle, q, lengths, table, out, workspace, row_start, most_rows, scale,
                                          error, stream)


class KV4Cache:
    """A paged 4-bit KV cache over tensors of the caller: k and v
    [blocks][kv_heads][block_size][head_dim / 2] uint8, k_scale and v_scale
    [blocks][kv_heads][block_size][head_dim / 64][2] float16, scale and low of
    each group of 64 values (fyb_kv4_cache)."""

    def __init__(self, k, v, k_scale, v_scale):
        import torch
        if k.dim() != 4 or k.shape != v.shape or k_scale.shape != (*k.shape[:3], k.shape[3] // 32, 2) or \
                v_scale.shape != k_scale.shape:
            raise ValueError("k, v: [blocks][kv_heads][block_size][head_dim / 2]; scales [blocks][kv_heads][block_size]"
                             "[head_dim / 64][2]")
        for name, t, kind in (("k", k, torch.uint8), ("v", v, torch.uint8), ("k_scale", k_scale, torch.float16),
                              ("v_scale", v_scale, torch.float16)):
            if t.dtype is not kind or not t.is_cuda or not t.is_contiguous() or t.device != k.device:
                raise ValueError("%s has to be a contiguous %s tensor on the cache's GPU" % (name, kind))
        self.tensors = k, v, k_scale, v_scale
        blocks, self.kv_heads, self.block_size, half = k.shape
        self.head_dim = 2 * half
        self._held = KV4Handle(KV4CacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), blocks,
                                            self.kv_heads, self.block_size, self.head_dim), k.get_device())
        self.desc, self._handle = self._held.cache, C.addressof(self._held)

    @classmethod
    def empty(cls, blocks, kv_heads, block_size, head_dim, device="cuda"):
        """A cache of its own tensors."""
        import torch
        k, v = (torch.zeros((blocks, kv_heads, block_size, head_dim // 2), dtype=torch.uint8, device=device)
                for _ in range(2))
        return cls(k, v, *(torch.zeros((blocks, kv_heads, block_size, head_dim // 64, 2), dtype=torch.float16,
                                       device=device) for _ in range(2)))

    def append(self, k, v, slots, positions=None, cos=None, sin=None, layout="interleaved", q=None, q_out=None,
               error=None, stream=None):
        """Store K and V rows [rows][kv_heads][head_dim] at slots[row], no slot
        twice (fyb_kv4_append). With cos / sin K is rotated to positions[row]
        first, and q to q_out in the same call."""
        (_native or _bind_tensors()).append4(self._handle, k, v, slots, positions, cos, sin, layout, q, q_out, error, stream)

    def read(self, slots, k_out, v_out, error=None, stream=None):
        """The values held at slots into k_out, v_out [len(slots)][kv_heads][head_dim] float32 (fyb_kv4_read)."""
        (_native or _bind_tensors()).read4(self._handle, slots, k_out, v_out, error, stream)

    def attention_workspace(self, requests, most_rows, heads):
        """A zeroed workspace for attention() calls of this size (one for each stream that calls)."""
        import torch
        need = lib.fyb_kv4_attention_workspace(requests, most_rows, heads, self.kv_heads, self.head_dim)
        if not need:
            raise ValueError("no attention of %d requests, %d rows, %d heads over %d KV heads of %d" %
                             (requests, most_rows, heads, self.kv_heads, self.head_dim))
        return torch.zeros(need, dtype=torch.uint8, device=self.tensors[0].device)

    def attention(self, q, lengths, table, out, workspace, row_start=None, most_rows=1, scale=None, error=None,
                  stream=None):
        """KV8Cache.attention over this cache (fyb_kv4_attention)."""
        (_native or _bind_tensors()).attention4(self._handle, q, lengths, table, out, workspace, row_start, most_rows, scale,
                                           error, stream)


def logprobs_workspace(rows, vocabulary, top=0, device="cuda"):
    """A zeroed workspace for logprobs() calls of this size (one for each stream that calls)."""
    import torch
    need = lib.fyb_logprobs_workspace(rows, vocabulary, top) if min(rows, vocabulary, top) >= 0 else 0
    if not need:
        raise ValueError("no log probabilities of %d rows of %d with %d alternatives" % (rows, vocabulary, top))
    return torch.zeros(need, dtype=torch.uint8, device=device)


def logprobs(logits, tokens, logprob, entropy, rank, top_tokens, top_logprobs, workspace, error=None, stream=None):
    """Of each row of logits [rows][vocabulary]: log probability and rank of
    tokens[row], entropy, and the most probable tokens with their log
    probabilities (fyb_logprobs). tokens and rank int32, logprob and entropy
    float32 [rows]; top_tokens int32 and top_logprobs float32 [rows][top]; any
    output may be None (tokens with logprob and rank, top_tokens with
    top_logprobs)."""
    (_native or _bind_tensors()).logprobs(logits, tokens, logprob, entropy, rank, top_tokens, top_logprobs, workspace, error,
                                     stream)


# ---------------------------------------------------------------- provider
IPC_HANDLE_BYTES = 64  # FYB_IPC_HANDLE_BYTES


def tp_exchange(handle, group=None):
    """Gather every rank's exchange-region handle in rank order through a
    torch.distributed group (any backend): the host side of connecting a
    tensor-parallel plan."""
    import torch.distributed as dist
    out = [None] * dist.get_world_size(group)
    dist.all_gather_object(out, bytes(handle), group=group)
    if any(h is None or len(h) != IPC_HANDLE_BYTES for h in out):
        raise ValueError("a rank has no exchange-region handle")
    return out


def tp_connect_all(plan, group=None):
    """Connect one rank's shard plan with every other rank's, or none of them.

    Every rank calls this with its plan (None when its plan_create declined).
    Returns True when all ranks opened all exchange regions. When any rank
    has no plan or no handle, no rank connects; when any rank fails to open
    the regions, the ranks that succeeded disconnect again. In both cases
    every rank returns False and its plan declines its steps (-1) without
    launching anything that would wait for the failed rank."""
    import torch.distributed as dist
    world = dist.get_world_size(group)
    handle = plan.tp_handle() if plan is not None else None
    handles = [None] * world
    dist.all_gather_object(handles, bytes(handle) if handle is not None else None, group=group)
    if any(h is None or len(h) != IPC_HANDLE_BYTES for h in handles):
        return False
    ok = plan.tp_connect(handles) == 0
    oks = [None] * world
    dist.all_gather_object(oks, ok, group=group)
    if not all(oks):
        if ok:
            plan.tp_disconnect()
        return False
    return True


class Provider:
    """A provider context: what nya_compute_create_for("cuda") owns.

    Plans must be freed before their context (backend/include/compute.h:6-8);
    close() frees any plan still alive first."""

    def __init__(self):
        import weakref
        self.api = api()
        self.state = self.api.create()
        if not self.state:
            raise RuntimeError("the B200 provider declined (no sm_100 device visible)")
        self._plans = weakref.WeakSet()

    def active(self):
        return bool(self.api.active(self.state))

    def matvec(self, weights, rows, cols, type_id, x):
        y = np.empty(rows, np.float32)
        r = self.api.matvec(self.state, _ptr(weights), rows, cols, type_id, _ptr(x), _ptr(y))
        return y if r == 0 else None

    def matmul(self, weights, rows, cols, type_id, x, batch):
        y = np.empty((batch, rows), np.float32)
        r = self.api.matmul(self.state, _ptr(weights), rows, cols, type_id, _ptr(x), _ptr(y), batch)
        return y if r == 0 else None

    def plan(self, model, capacity):
        p = self.api.plan_create(self.state, C.c_void_p(model.ptr), capacity)
        if not p:
            return None
        plan = Plan(self, p, model)
        self._plans.add(plan)
        return plan

    def close(self):
        if self.state:
            for plan in list(self._plans):
                plan.close()
            self.api.destroy(self.state)
            self.state = None

    def __del__(self):
        self.close()


class Batch:
    """B sequences (1..16) of one plan's model decoded together (fyb_batch_*):
    each sequence has its own KV cache and position; every projection reads
    each weight once per step for all of them. A plan that is closed frees its
    batches, which then refuse every step.

    kv "int8" or "e4m3": a paged 8-bit cache of `blocks` blocks of block_size
    tokens that the sequences share, instead of an fp16 cache of the plan's
    capacity each (fyb_batch_create_kv8); "uint4": one in 4 bits
    (fyb_batch_create_kv4)."""

    _ptr = None  # until it is made, and where it is declined

    def __init__(self, plan, batch, kv=None, blocks=0, block_size=32):
        self.plan, self.B = plan, batch
        self.V = plan.model.vocabulary
        if kv is None:
            ptr = lib.fyb_batch_create(C.c_void_p(plan.ptr), batch)
        elif kv == "uint4":
            ptr = lib.fyb_batch_create_kv4(C.c_void_p(plan.ptr), batch, blocks, block_size)
        else:
            ptr = lib.fyb_batch_create_kv8(C.c_void_p(plan.ptr), batch, blocks, block_size, _format(kv))
        if not ptr:
            raise ValueError("batch of %d declined" % batch)
        self._ptr = ptr
        plan._batches.add(ptr)

    @property
    def ptr(self):
        """The batch, or None once it or its plan is closed."""
        return self._ptr if self._ptr and self._ptr in self.plan._batches else None

    def _req(self, tokens, positions):
        t = np.ascontiguousarray(tokens, np.uint32)
        p = np.ascontiguousarray(positions, np.uint32)
        assert t.shape == (self.B,) and p.shape == (self.B,)
        return t, p

    def step(self, tokens, positions, logits=True):
        """One step: (logits [B][V] or None, argmax [B])."""
        t, p = self._req(tokens, positions)
        lg = np.empty((self.B, self.V), np.float32) if logits else None
        am = np.empty(self.B, np.uint32)
        r = lib.fyb_batch_step(C.c_void_p(self.ptr), _ptr(t), _ptr(p), _ptr(lg), _ptr(am))
        if r:
            raise RuntimeError("fyb_batch_step failed (%d)" % r)
        return lg, am

    def score(self, tokens, positions, targets=None, top=0):
        """One step whose logits stay on the device (fyb_batch_score): dict of
        logprob, rank (with targets, the tokens that follow; negative: none),
        entropy [B], top_tokens and top_logprobs [B][top]."""
        t, p = self._req(tokens, positions)
        if not 0 <= top <= 32:
            raise ValueError("top is 0 to 32")
        out = dict(entropy=np.empty(self.B, np.float32), top_tokens=np.empty((self.B, top), np.int32),
                   top_logprobs=np.empty((self.B, top), np.float32))
        if targets is not None:
            targets = np.ascontiguousarray(targets, np.int32)
            if targets.shape != (self.B,):
                raise ValueError("targets has to have one token for each sequence")
            out |= dict(logprob=np.empty(self.B, np.float32), rank=np.empty(self.B, np.int32))
        r = lib.fyb_batch_score(C.c_void_p(self.ptr), _ptr(t), _ptr(p), _ptr(targets), _ptr(out.get("logprob")),
                                _ptr(out.get("rank")), _ptr(out["entropy"]), top, _ptr(out["top_tokens"]),
                                _ptr(out["top_logprobs"]))
        if r:
            raise RuntimeError("fyb_batch_score failed (%d)" % r)
        return out

    def decode_greedy(self, tokens, positions, steps):
        """Greedy tokens [steps][B] decoded on the device."""
        t, p = self._req(tokens, positions)
        out = np.empty((steps, self.B), np.uint32)
        r = lib.fyb_batch_decode_greedy(C.c_void_p(self.ptr), _ptr(t), _ptr(p), steps, _ptr(out))
        if r:
            raise RuntimeError("fyb_batch_decode_greedy failed (%d)" % r)
        return out

    def time_greedy(self, tokens, positions, steps):
        """Milliseconds per greedy step (device events)."""
        t, p = self._req(tokens, positions)
        return lib.fyb_batch_time_greedy(C.c_void_p(self.ptr), _ptr(t), _ptr(p), steps)

    def free_blocks(self):
        """Blocks of a paged batch that no sequence holds."""
        return lib.fyb_batch_free_blocks(C.c_void_p(self.ptr))

    def launches_per_step(self):
        return lib.fyb_batch_launches_per_step(C.c_void_p(self.ptr))

    def close(self):
        if self.ptr:
            self.plan._batches.remove(self._ptr)
            lib.fyb_batch_free(C.c_void_p(self._ptr))
        self._ptr = None

    def __del__(self):
        self.close()


class Plan:
    """A resident plan (nya_compute_plan)."""

    def __init__(self, provider, ptr, model):
        self.provider, self.ptr, self.model = provider, ptr, model
        self.api = provider.api
        self.logits = np.empty(model.vocabulary, np.float32)
        self._batches = set()  # alive; freed with the plan, in whatever order Python collects the two

    def token(self, token, position, logits=True):
        out = self.logits if logits else None
        r = self.api.plan_token(self.ptr, token, position, 1 if logits else 0, _ptr(out))
        return r

    def prefill(self, tokens, position):
        tokens = np.ascontiguousarray(tokens, np.uint32)
        return self.api.plan_prefill(self.ptr, _ptr(tokens), len(tokens), position, _ptr(self.logits))

    def stats(self):
        s = ComputeStats()
        self.api.plan_stats(self.ptr, C.byref(s))
        return s.as_dict()

    def read_kv(self, layer, position, count):
        width = self.model.kv_dim
        k = np.empty((count, width), np.float32)
        v = np.empty((count, width), np.float32)
        r = self.api.plan_read_kv(self.ptr, layer, position, count, _ptr(k), _ptr(v), count * width)
        return (k, v) if r == 0 else None

    def verify(self, tokens, position):
        """Logits [k][V] of k draft tokens at positions position.. (one pass)."""
        t = np.ascontiguousarray(tokens, np.uint32)
        out = np.empty((len(t), self.model.vocabulary), np.float32)
        r = lib.fyb_plan_verify(C.c_void_p(self.ptr), _ptr(t), len(t), position, _ptr(out))
        return out if r == 0 else None

    def decode_greedy(self, token, position, steps):
        out = np.empty(steps, np.uint32)
        r = lib.fyb_plan_decode_greedy(C.c_void_p(self.ptr), token, position, steps, _ptr(out))
        return out if r == 0 else None

    def time_greedy(self, token, position, steps):
        return lib.fyb_plan_time_greedy(C.c_void_p(self.ptr), token, position, steps)

    def launches_per_token(self):
        return lib.fyb_plan_launches_per_token(C.c_void_p(self.ptr))

    def decode_form(self):
        """0 per-operation kernels, 1 the persistent decode kernel."""
        return lib.fyb_plan_decode_form(C.c_void_p(self.ptr))

    def tp_info(self):
        """(rank, size) of the plan's tensor-parallel shard."""
        r, n = C.c_uint(0), C.c_uint(0)
        lib.fyb_plan_tp_info(C.c_void_p(self.ptr), C.byref(r), C.byref(n))
        return r.value, n.value

    def tp_handle(self):
        """This rank's exchange-region handle (bytes), or None."""
        buf = C.create_string_buffer(IPC_HANDLE_BYTES)
        if lib.fyb_plan_tp_handle(C.c_void_p(self.ptr), buf, IPC_HANDLE_BYTES) != 0:
            return None
        return buf.raw

    def tp_connect(self, handles):
        """Open the other ranks' regions; handles: one bytes object per rank, in rank order."""
        blob = b"".join(handles)
        return lib.fyb_plan_tp_connect(C.c_void_p(self.ptr), C.c_char_p(blob), len(handles))

    def tp_disconnect(self):
        """Decline every later step without launching (another rank failed)."""
        return lib.fyb_plan_tp_disconnect(C.c_void_p(self.ptr))

    def tp_connect_local(self, plans):
        """Connect this plan to the other shard plans of this process
        (plans: every rank's Plan, in rank order)."""
        arr = (C.c_void_p * len(plans))(*[q.ptr for q in plans])
        return lib.fyb_plan_tp_connect_local(C.c_void_p(self.ptr), arr, len(plans))

    def error(self):
        """The device error word: 0 none, 1 a bounded wait ran out, 2 non-finite
        logits, 4 an index out of range."""
        return lib.fyb_plan_error(C.c_void_p(self.ptr))

    def trace(self, token, position, detail=False):
        """Per-CTA trace points of one persistent decode step: array
        [points][grid] of globaltimer nanoseconds (start, then per layer the
        ends of QKV, attention, O, gate/up and down, the end of the logits,
        exit), or None. With detail=True, a pair (that array, per-warp
        records of layer layers // 2 [grid][16][32], decode_kernel.cuh)."""
        grid = C.c_uint(0)
        L = self.model.config.layers
        points = 1 + 5 * L + 2
        n = points * 1024
        out = np.zeros(n, np.uint64)
        wn = 1024 * 16 * 32
        wout = np.zeros(wn, np.uint64) if detail else None
        r = lib.fyb_plan_trace(C.c_void_p(self.ptr), token, position, _ptr(out), n, C.byref(grid),
                               _ptr(wout) if detail else None, wn if detail else 0)
        if r < 0:
            return None
        cta = out[: r * grid.value].reshape(r, grid.value)
        if not detail:
            return cta
        return cta, wout[: grid.value * 16 * 32].reshape(grid.value, 16, 32)

    def profile(self, token, position, steps):
        """Per-class milliseconds of one decode step: matrix, attention, other."""
        out = np.zeros(3, np.float64)
        r = lib.fyb_plan_profile(C.c_void_p(self.ptr), token, position, steps, _ptr(out))
        return out if r == 0 else None

    def time_projection(self, layer, which, reps):
        """(ms per launch, algorithmic bytes) of one fused projection kernel."""
        nbytes = C.c_size_t()
        ms = lib.fyb_plan_time_projection(C.c_void_p(self.ptr), layer, which, reps, C.byref(nbytes))
        return ms, nbytes.value

    def close(self):
        if self.ptr:
            while self._batches:
                lib.fyb_batch_free(C.c_void_p(self._batches.pop()))
            self.api.plan_free(self.ptr)
            self.ptr = None

    def __del__(self):
        self.close()
