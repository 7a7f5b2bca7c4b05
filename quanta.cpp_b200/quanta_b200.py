"""Python host mirror of the engine's C ABI (include/quanta_b200.h), via ctypes.

The names follow the reference's C++ interface (engine/src/model.h, ops.h, sampler.h, session.h):
    Model(path, ctx).forward(token, pos, hq) / forward_batch(tokens, pos0, hq) / head(hq) / last_head_rows
    quantize_q8(x) ; DeviceTensor(dtype, rows, cols, raw).matvec(q, d, r0, r1) / .matmul(...)
    Model.generate(prompt, SamplerParams(...), shortlist=True, batch_prefill=True, n_gen=64)
    PagedKV.empty(...).reserve / append / attention / read / fork / reorder / free / compact  the paged 8-bit KV cache (torch)
    rms_norm_q8(x, weight, residual=r), dequantize_q8(q, d), Rope(...)(q, k, positions)  around a layer's products (torch)
    BeamSelector(k)(logits, scores)  the selection of a beam search's next step (torch)
    synth_model(path, ...)  seeded random-init .qnt writer
There is no CPU fallback: importing works anywhere, but every call needs libquanta_b200.so and a GPU, and fails
loudly when either is missing.
"""
from __future__ import annotations

import ctypes as C
import math
import os
from dataclasses import dataclass
from pathlib import Path

import numpy as np

PKG = Path(__file__).resolve().parent
LIB_DIR = Path(os.environ["QNT_LIB_DIR"]) if os.environ.get("QNT_LIB_DIR") else PKG / "lib"  # timeline.py: lib_stamps

F32, F16, Q8_0, Q4_0 = 0, 1, 2, 3
BF16 = 4  # activations only: the paged KV cache, norm, rope and beams
QK = 32
GEN_SHORTLIST, GEN_BATCH_PREFILL = 1, 2


class QntError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"quanta_b200 error {code}: {msg}")
        self.code = code


class HeadQuery(C.Structure):
    _fields_ = [("top_k", C.c_int), ("n_valid", C.c_int), ("must", C.POINTER(C.c_int)), ("n_must", C.c_int)]


class HParams(C.Structure):
    _fields_ = [(n, C.c_int) for n in "vocab_size dim n_layers n_heads n_kv_heads head_dim ffn_dim max_seq".split()] + [
        ("rope_theta", C.c_float), ("norm_eps", C.c_float), ("tied_embeddings", C.c_int), ("qkv_bias", C.c_int),
        ("flags", C.c_uint32), ("n_tokens", C.c_int), ("ctx_len", C.c_int), ("has_shortlist", C.c_int)]


class SamplerParamsC(C.Structure):
    _fields_ = [("temperature", C.c_float), ("top_k", C.c_int), ("top_p", C.c_float), ("min_p", C.c_float),
                ("repeat_penalty", C.c_float), ("repeat_window", C.c_int), ("seed", C.c_uint64)]


class GenStatsC(C.Structure):
    _fields_ = [("prefill_ms", C.c_double), ("decode_ms", C.c_double), ("head_rows", C.c_longlong),
                ("head_calls", C.c_longlong), ("kernels_per_step", C.c_int)]


class SynthCfg(C.Structure):
    _fields_ = [(n, C.c_int) for n in "vocab_size dim n_layers n_heads n_kv_heads head_dim ffn_dim max_seq".split()] + [
        ("rope_theta", C.c_float), ("norm_eps", C.c_float)] + [(n, C.c_int) for n in "mlp_q4 q4_group shortlist n_tokens".split()] + [
        ("w_std", C.c_float), ("seed", C.c_uint64), ("n_threads", C.c_int), ("flags", C.c_uint32),
        ("tok_blob", C.c_char_p), ("tok_len", C.c_uint64)]


class KVCacheC(C.Structure):
    _fields_ = [(n, C.c_int) for n in "n_layers n_kv_heads head_dim page_tokens n_pages max_seqs max_pages".split()] + [
        (n, C.c_void_p) for n in "codes scales refs table lens status".split()]


@dataclass
class SamplerParams:
    """engine/src/sampler.h:9-18 defaults (Qwen2.5-Instruct generation config)."""
    temperature: float = 0.7
    top_k: int = 20
    top_p: float = 0.8
    min_p: float = 0.0
    repeat_penalty: float = 1.1
    repeat_window: int = 0
    seed: int = 0


_lib = None
_synth = None


def lib_path() -> Path:
    return LIB_DIR / "libquanta_b200.so"


def lib() -> C.CDLL:
    """Loads libquanta_b200.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        p = lib_path()
        if not p.exists():
            raise RuntimeError(f"{p} is missing: run `python quanta.cpp_b200/build.py` (nvcc, sm_100a)")
        L = C.CDLL(str(p))
        P, I, F = C.c_void_p, C.c_int, C.c_float
        L.qnt_last_error.restype = C.c_char_p
        L.qnt_tensor_upload.argtypes = [I, I, I, P, C.POINTER(P)]
        L.qnt_tensor_free.argtypes = [P]
        L.qnt_quantize_q8.argtypes = [P, I, I, P, P, P]
        L.qnt_matvec.argtypes = [P, P, P, I, I, P, P]
        L.qnt_matmul.argtypes = [P, P, P, I, I, I, P, I, I, P]
        L.qnt_ops_check.argtypes = [P]
        L.qnt_quantize_q8_host.argtypes = [P, I, P, P]
        L.qnt_matvec_host.argtypes = [P, P, P, I, I, P]
        L.qnt_matmul_host.argtypes = [P, P, P, I, I, I, P, I, I]
        L.qnt_model_open.argtypes = [C.c_char_p, I, I, C.POINTER(P)]
        L.qnt_model_close.argtypes = [P]
        L.qnt_model_close.restype = None
        L.qnt_model_hparams.argtypes = [P, C.POINTER(HParams)]
        L.qnt_model_forward.argtypes = [P, I, I, C.POINTER(HeadQuery), P]
        L.qnt_model_forward_batch.argtypes = [P, P, I, I, C.POINTER(HeadQuery), P]
        L.qnt_model_head.argtypes = [P, C.POINTER(HeadQuery), P, P, P]
        L.qnt_model_last_head_rows.argtypes = [P]
        L.qnt_model_has_shortlist.argtypes = [P]
        L.qnt_model_kv_cache_bytes.argtypes = [P]
        L.qnt_model_kv_cache_bytes.restype = C.c_size_t
        L.qnt_model_weight_bytes.argtypes = [P]
        L.qnt_model_weight_bytes.restype = C.c_size_t
        L.qnt_export_device_layout.argtypes = [C.c_char_p, C.c_char_p]
        L.qnt_model_packed_tensors.argtypes = [P]
        L.qnt_generate.argtypes = [P, P, I, C.POINTER(SamplerParamsC), I, I, P, C.POINTER(GenStatsC)]
        L.qnt_set_device.argtypes = [I]
        L.qnt_session_begin.argtypes = [P, P, I, C.POINTER(SamplerParamsC), I]
        L.qnt_session_step.argtypes = [P, I]
        L.qnt_session_read.argtypes = [P, P, I, C.POINTER(GenStatsC)]
        L.qnt_model_stream.argtypes = [P]
        L.qnt_model_stream.restype = P
        L.qnt_batch_init.argtypes = [P, I, I]
        L.qnt_prefill_batch.argtypes = [P, I, P, I, C.POINTER(I)]
        L.qnt_decode_batch.argtypes = [P, P, P, I, P]
        L.qnt_batch_reset.argtypes = [P, I]
        L.qnt_batch_init_paged.argtypes = [P, I, I, I, I]
        L.qnt_batch_fork.argtypes = [P, I, I]
        L.qnt_batch_resize.argtypes = [P, I]
        L.qnt_beam_search.argtypes = [P, P, I, I, I, I, P, P, P]
        L.qnt_sampler_create.argtypes = [C.POINTER(SamplerParamsC), C.POINTER(P)]
        L.qnt_sampler_sample.argtypes = [P, P, I, P, I, C.POINTER(I), P]
        L.qnt_sampler_free.argtypes = [P]
        L.qnt_sampler_free.restype = None
        L.qnt_bench_mma_i8.argtypes = [I, C.POINTER(C.c_double)]
        L.qnt_wait_probe.argtypes = [C.c_uint, P]
        L.qnt_session_feed.argtypes = [P, P, I]
        L.qnt_model_nll.argtypes = [P, P, I, C.POINTER(C.c_double)]
        L.qnt_session_rewind.argtypes = [P, I]
        L.qnt_session_last.argtypes = [P, C.POINTER(I), C.POINTER(I)]
        L.qnt_tokenizer_open.argtypes = [C.c_char_p, C.POINTER(P)]
        L.qnt_tokenizer_free.argtypes = [P]
        L.qnt_tokenizer_free.restype = None
        L.qnt_tokenizer_n_tokens.argtypes = [P]
        L.qnt_tokenize.argtypes = [P, C.c_char_p, C.c_size_t, P, I]
        L.qnt_token_piece.argtypes = [P, I, C.c_char_p, I]
        L.qnt_token_id.argtypes = [P, C.c_char_p]
        L.qnt_sampler_sample_noalloc.argtypes = [C.POINTER(SamplerParamsC), C.POINTER(C.c_uint64), P, I, P, I,
                                                 C.POINTER(I), P]
        K, Z, LL = C.POINTER(KVCacheC), C.c_size_t, C.c_longlong
        L.qnt_kv_page_workspace.argtypes = [K]
        L.qnt_kv_page_workspace.restype = Z
        L.qnt_kv_reserve.argtypes = [K, P, P, I, P, Z, P]
        L.qnt_kv_fork.argtypes = [K, P, P, I, P, Z, P]
        L.qnt_kv_reorder_workspace.argtypes = [K]
        L.qnt_kv_reorder_workspace.restype = Z
        L.qnt_kv_reorder.argtypes = [K, P, P, I, I, P, Z, P]
        L.qnt_kv_free.argtypes = [K, P, I, P]
        L.qnt_kv_compact.argtypes = [K, P, Z, P]
        L.qnt_kv_copy.argtypes = [K, P, P, I, P]
        L.qnt_kv_append.argtypes = [K, I, P, P, I, LL, LL, P, P, I, I, I, P]
        L.qnt_kv_read.argtypes = [K, I, P, P, P, I, I, P, P, I, P]
        L.qnt_kv_attention_workspace.argtypes = [K, I, I, I, I, I]
        L.qnt_kv_attention_workspace.restype = Z
        L.qnt_kv_attention.argtypes = [K, I, P, I, LL, I, P, P, I, I, I, I, F, I, P, P, P, Z, P]
        L.qnt_kv_check.argtypes = [K, P]
        L.qnt_rms_norm_q8.argtypes = [P, I, LL, P, I, LL, P, F, I, I, P, P, P]
        L.qnt_dequantize_q8.argtypes = [P, P, I, I, P, I, P]
        L.qnt_rope.argtypes = [P, LL, P, LL, I, P, LL, P, LL, I, I, I, I, I, P, F, P, I, P]
        L.qnt_beam_workspace.argtypes = [I, I, I, I]
        L.qnt_beam_workspace.restype = Z
        L.qnt_beam_select.argtypes = [P, I, LL, P, P, I, I, I, I, I, P, P, P, P, Z, P]
        _lib = L
    return _lib


def _check(rc: int) -> int:
    if rc < 0:
        raise QntError(rc, lib().qnt_last_error().decode(errors="replace"))
    return rc


def _ptr(a: np.ndarray | None):
    return None if a is None else a.ctypes.data_as(C.c_void_p)


def exported_symbols() -> list[str]:
    """Every function declared in include/quanta_b200.h."""
    import re
    hdr = (PKG.parent / "include" / "quanta_b200.h").read_text()
    return sorted(set(re.findall(r"^\w[\w\s\*]*?\b(qnt_\w+)\s*\(", hdr, re.M)))


def device_count() -> int:
    return lib().qnt_device_count()


def set_device(d: int) -> None:
    _check(lib().qnt_set_device(d))


# ---------------------------------------------------------------- ops level

def quantize_q8(x: np.ndarray):
    """quantize_q8 (engine/src/ops_ref.cpp:69-83) on the device: returns (q int8[n], d f32[n/32])."""
    x = np.ascontiguousarray(x, np.float32)
    q = np.empty(x.size, np.int8)
    d = np.empty(x.size // QK, np.float32)
    _check(lib().qnt_quantize_q8_host(_ptr(x), x.size, _ptr(q), _ptr(d)))
    return q, d


class DeviceTensor:
    """A quantized matrix in HBM (the .qnt byte layout in, device copy inside)."""

    def __init__(self, dtype: int, rows: int, cols: int, raw: np.ndarray | bytes):
        buf = np.frombuffer(raw, np.uint8) if isinstance(raw, (bytes, bytearray)) else np.ascontiguousarray(raw).view(np.uint8)
        self.dtype, self.rows, self.cols = dtype, rows, cols
        self._buf = buf
        h = C.c_void_p()
        _check(lib().qnt_tensor_upload(dtype, rows, cols, _ptr(buf), C.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.qnt_tensor_free(self.h)
        self.h = None

    __del__ = close

    def matvec(self, q: np.ndarray, d: np.ndarray, r0: int = 0, r1: int | None = None) -> np.ndarray:
        r1 = self.rows if r1 is None else r1
        out = np.zeros(self.rows, np.float32)
        _check(lib().qnt_matvec_host(self.h, _ptr(np.ascontiguousarray(q, np.int8)), _ptr(np.ascontiguousarray(d, np.float32)),
                                     r0, r1, _ptr(out)))
        return out

    def matmul(self, q: np.ndarray, d: np.ndarray, r0: int = 0, r1: int | None = None, impl: int = 0) -> np.ndarray:
        """q [n][cols] int8, d [n][cols/32] -> out [n][rows] (rows outside [r0, r1) are 0)."""
        r1 = self.rows if r1 is None else r1
        q = np.ascontiguousarray(q, np.int8)
        n = q.shape[0]
        out = np.zeros((n, self.rows), np.float32)
        _check(lib().qnt_matmul_host(self.h, _ptr(q), _ptr(np.ascontiguousarray(d, np.float32)), n, r0, r1, _ptr(out),
                                     self.rows, impl))
        return out



class Sampler:
    """Sampler (engine/src/sampler.h:20-38) on the device: sample(logits, n_valid, history) -> id, as
    Sampler::sample (sampler.cpp:22-85).  `logits` is a float32 CUDA tensor (torch) on the current device and is edited
    in place like the reference's array; `history` is a sequence of ids."""

    def __init__(self, sp: SamplerParams):
        spc = SamplerParamsC(sp.temperature, sp.top_k, sp.top_p, sp.min_p, sp.repeat_penalty, sp.repeat_window, sp.seed)
        h = C.c_void_p()
        _check(lib().qnt_sampler_create(C.byref(spc), C.byref(h)))
        self.h = h
        self.params = sp

    def sample(self, logits, n_valid: int | None = None, history=(), stream=None) -> int:
        if not (getattr(logits, "is_cuda", False) and str(logits.dtype) == "torch.float32" and logits.is_contiguous()):
            raise TypeError("logits must be a contiguous float32 CUDA tensor")
        n_valid = logits.numel() if n_valid is None else n_valid
        hist = np.ascontiguousarray(np.asarray(history, np.int32).ravel())
        tok = C.c_int(-1)
        st = None if stream is None else C.c_void_p(stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream))
        _check(lib().qnt_sampler_sample(self.h, C.c_void_p(logits.data_ptr()), n_valid, _ptr(hist) if hist.size else None,
                                        hist.size, C.byref(tok), st))
        return tok.value

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.qnt_sampler_free(self.h)
        self.h = None

    __del__ = close


def sample_noalloc(sp: SamplerParams, rng_state: int, logits, n_valid: int | None = None, history=(), stream=None):
    """qnt_sampler_sample_noalloc: the Sampler without an object and without allocating (static device scratch).
    rng_state is the xorshift64* state ((seed or any nonzero) | 1 to start); returns (id, next rng_state)."""
    if not (getattr(logits, "is_cuda", False) and str(logits.dtype) == "torch.float32" and logits.is_contiguous()):
        raise TypeError("logits must be a contiguous float32 CUDA tensor")
    n_valid = logits.numel() if n_valid is None else n_valid
    spc = SamplerParamsC(sp.temperature, sp.top_k, sp.top_p, sp.min_p, sp.repeat_penalty, sp.repeat_window, sp.seed)
    hist = np.ascontiguousarray(np.asarray(history, np.int32).ravel())
    state = C.c_uint64(rng_state)
    tok = C.c_int(-1)
    st = None if stream is None else C.c_void_p(stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream))
    _check(lib().qnt_sampler_sample_noalloc(C.byref(spc), C.byref(state), C.c_void_p(logits.data_ptr()), n_valid,
                                            _ptr(hist) if hist.size else None, hist.size, C.byref(tok), st))
    return tok.value, state.value


class PagedKV:
    """The paged 8-bit KV cache (qnt_kv_*): many sequences in pages of one pool, int8 codes with a f32 scale for each block
    of 16 tokens, K or V, layer and kv head.  The arrays are torch CUDA tensors that the caller may keep and look at:
        codes  int8 [n_pages, n_layers, 2, n_kv_heads, page_tokens * head_dim]  (K tile [head_dim/16][page_tokens][16
               dims], V tile [page_tokens/16][head_dim][16 tokens])
        scales float32 [n_pages, n_layers, 2, n_kv_heads, page_tokens / 16]
        refs int32 [n_pages], table int32 [max_seqs, max_pages], lens int32 [max_seqs]
    Sequence lists (seqs, starts, extra, ...) are contiguous int32 CUDA tensors: tokens starts[j] .. starts[j + 1] - 1 of a
    call belong to sequence seqs[j].  Work is queued on `stream` (a torch stream or a cudaStream_t's number; default: torch's
    current stream), nothing waits.  With another stream than the current one a call is as if made within torch.cuda.stream(stream):
    its outputs belong to that stream, and what it reads has to be ready there.  Errors that kernels find (no free pages, a
    sequence out of range) are raised by check().  Calls that write the cache must be ordered against its other calls; the
    object's workspaces are one per stream, and live as long as the object: a graph that captured calls is replayed while the
    object exists, ordered against the calls on the stream that it was captured on."""

    def __init__(self, codes, scales, refs, table, lens):
        import torch
        self._torch = torch
        i32 = torch.int32
        for name, t, dt, dim in (("codes", codes, torch.int8, 5), ("scales", scales, torch.float32, 5), ("refs", refs, i32, 1),
                                 ("table", table, i32, 2), ("lens", lens, i32, 1)):
            if not (t.is_cuda and t.dtype == dt and t.dim() == dim and t.is_contiguous() and t.device == codes.device):
                raise TypeError(f"{name} must be a contiguous {dim}-dimensional {dt} CUDA tensor on the codes' device")
        n_pages, n_layers, two, n_kv, tile = codes.shape
        page_tokens = scales.shape[4] * 16
        if two != 2 or scales.shape[:4] != codes.shape[:4] or refs.shape[0] != n_pages or lens.shape[0] != table.shape[0] \
                or page_tokens == 0 or tile % page_tokens:
            raise ValueError("codes, scales, refs, table and lens do not describe one cache")
        self.codes, self.scales, self.refs, self.table, self.lens = codes, scales, refs, table, lens
        self.n_layers, self.n_kv_heads, self.head_dim, self.page_tokens = n_layers, n_kv, tile // page_tokens, page_tokens
        self.device = codes.device
        self._status = torch.zeros(1, dtype=i32, device=self.device)
        self._c = KVCacheC(n_layers, n_kv, self.head_dim, page_tokens, n_pages, table.shape[0], table.shape[1], codes.data_ptr(),
                           scales.data_ptr(), refs.data_ptr(), table.data_ptr(), lens.data_ptr(), self._status.data_ptr())
        self._p = C.byref(self._c)
        self._types = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
        self._ws, self._kept, self._need, self._i32, self._reorder_ws = {}, [], {}, i32, None
        self._lib, self._index = lib(), codes.device.index  # a call's host time counts where few tokens are decoded
        self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        self._current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
        self._page_ws = lib().qnt_kv_page_workspace(self._p)
        if self._page_ws == 0:
            raise QntError(-1, lib().qnt_last_error().decode(errors="replace"))

    @classmethod
    def empty(cls, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, max_seqs: int, max_pages: int,
              page_tokens: int = 64, device="cuda"):
        """A cache without sequences."""
        import torch
        z = dict(dtype=torch.int32, device=device)
        return cls(torch.zeros((n_pages, n_layers, 2, n_kv_heads, page_tokens * head_dim), dtype=torch.int8, device=device),
                   torch.zeros((n_pages, n_layers, 2, n_kv_heads, page_tokens // 16), dtype=torch.float32, device=device),
                   torch.zeros(n_pages, **z), torch.full((max_seqs, max_pages), -1, **z), torch.zeros(max_seqs, **z))

    def _stream(self, stream):
        if stream is None:
            return self._raw_stream(self._index) if self._raw_stream else self._torch.cuda.current_stream(self.device).cuda_stream
        return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)

    def _allocating_on(self, stream):
        """Within it torch allocates for work on this stream: from its own pool, whose memory no other stream still uses."""
        cuda = self._torch.cuda
        if not hasattr(stream, "cuda_stream"):
            stream = cuda.ExternalStream(int(stream), device=self.device) if int(stream) else cuda.default_stream(self.device)
        return cuda.stream(stream)

    def _workspace(self, stream: int, need: int):
        ws = self._ws.get(stream)
        if ws is None or ws.numel() < need:
            size = max(need, self._page_ws, 1 << 20)
            if ws is not None:  # the old one stays: queued kernels and captured graphs still write to it
                self._kept.append(ws)
                size = max(size, 2 * ws.numel())  # (all of the old ones together are less than the new one)
            with self._allocating_on(stream):
                ws = self._ws[stream] = self._torch.empty(size, dtype=self._torch.uint8, device=self.device)
        return ws.data_ptr(), ws.numel()

    def _run(self, call, *args):
        """A launching call of the library: on the cache's device, whichever is current."""
        if self._current_device() == self._index:
            rc = call(*args)
        else:
            with self._torch.cuda.device(self._index):
                rc = call(*args)
        if rc:
            _check(rc)

    def _list(self, *lists):
        for t in lists:
            if t.dtype is not self._i32 or t.get_device() != self._index or not t.is_contiguous():
                raise TypeError("sequence lists must be contiguous int32 CUDA tensors on the cache's device")
        return lists[0].numel()

    def _rows(self, name, x, heads=None):
        """The type and the token stride of rows [tokens, heads, head_dim]."""
        shape, st, hd = x.shape, x.stride(), self.head_dim
        dt = self._types.get(x.dtype)
        if not (len(st) == 3 and st[2] == 1 and st[1] == hd and shape[2] == hd and dt is not None and
                x.get_device() == self._index and (heads is None or shape[1] == heads)):
            raise TypeError(f"{name} must be a float32, float16 or bfloat16 CUDA tensor [tokens, heads, {self.head_dim}] on the "
                            "cache's device whose heads are contiguous within a token")
        return dt, st[0]

    def reserve(self, seqs, extra, stream=None):
        """lens[seqs] += extra, with the pages for it."""
        n = self._list(seqs, extra)
        if extra.numel() != n:
            raise ValueError("one extra per sequence")
        s = self._stream(stream)
        w, nb = self._workspace(s, self._page_ws)
        self._run(self._lib.qnt_kv_reserve, self._p, seqs.data_ptr(), extra.data_ptr(), n, w, nb, s)

    def fork(self, src, dst, stream=None):
        """Empty sequences dst become copies of src: full pages shared, a part-filled last page copied."""
        n = self._list(src, dst)
        if dst.numel() != n:
            raise ValueError("one dst per src")
        s = self._stream(stream)
        w, nb = self._workspace(s, self._page_ws)
        self._run(self._lib.qnt_kv_fork, self._p, src.data_ptr(), dst.data_ptr(), n, w, nb, s)

    def reorder(self, seqs, parents, group: int | None = None, stream=None):
        """A beam search's step: sequence seqs[i] becomes what seqs[i - i % group + parents[i]] was before the call (group: beams of a
        request, by default the whole list).  Full pages are shared; one child of each parent goes on with its part-filled last
        page, the others get copies of what it holds; pages that nothing uses any more are free again."""
        if stream is not None:
            with _on_stream(stream, self.device):
                return self.reorder(seqs, parents, group)
        if self._reorder_ws is None:
            self._reorder_ws = self._lib.qnt_kv_reorder_workspace(self._p)
        s = self._stream(None)
        ws = self._ws.get(s)
        if ws is None or ws.numel() < self._reorder_ws:
            self._workspace(s, self._reorder_ws)
            ws = self._ws[s]
        rc = (_torch_module or _torch_calls()).kv_reorder(C.addressof(self._c), seqs, parents, group, ws)
        if rc:
            _check(rc)

    def free(self, seqs, stream=None):
        """The sequences give back their pages and become empty."""
        self._run(self._lib.qnt_kv_free, self._p, seqs.data_ptr(), self._list(seqs), self._stream(stream))

    def compact(self, stream=None):
        """The pages in use move together to the lowest indices."""
        s = self._stream(stream)
        w, nb = self._workspace(s, self._page_ws)
        self._run(self._lib.qnt_kv_compact, self._p, w, nb, s)

    def copy_pages(self, src, dst, stream=None):
        """Codes and scales of pages src over those of pages dst, all layers."""
        n = self._list(src, dst)
        if dst.numel() != n:
            raise ValueError("one dst per src")
        self._run(self._lib.qnt_kv_copy, self._p, src.data_ptr(), dst.data_ptr(), n, self._stream(stream))

    def append(self, layer: int, k, v, seqs, starts, max_new: int | None = None, stream=None):
        """Quantizes rows k, v [tokens, n_kv_heads, head_dim] into a layer, as the last positions of their sequences
        (reserve first); max_new bounds a sequence's new tokens."""
        dt, ks = self._rows("k", k, self.n_kv_heads)
        vt, vs = self._rows("v", v, self.n_kv_heads)
        m = k.shape[0]
        if vt != dt or v.shape[0] != m:
            raise TypeError("k and v must have the same type and number of tokens")
        n = self._list(seqs, starts)
        if starts.numel() != n + 1:
            raise ValueError("starts must have one entry more than seqs")
        self._run(self._lib.qnt_kv_append, self._p, layer, k.data_ptr(), v.data_ptr(), dt, ks, vs, seqs.data_ptr(),
                  starts.data_ptr(), n, m, m if max_new is None else max_new, self._stream(stream))

    def read(self, layer: int, seqs, first, starts, n_tok: int, dtype=None, stream=None):
        """Values of positions first[j] + i of sequence seqs[j] as rows starts[j] + i: (K, V) [n_tok, n_kv_heads, head_dim]
        (float32 unless dtype says otherwise)."""
        t = self._torch
        dtype = dtype or t.float32
        if dtype not in self._types:
            raise TypeError("dtype must be float32, float16 or bfloat16")
        n = self._list(seqs, first, starts)
        if first.numel() != n or starts.numel() != n + 1:
            raise ValueError("one first per sequence, and one entry more in starts")
        shape = (n_tok, self.n_kv_heads, self.head_dim)
        if stream is None:
            k = self.scales.new_empty(shape, dtype=dtype)
            v = t.empty_like(k)
        else:
            with self._allocating_on(stream):
                k = self.scales.new_empty(shape, dtype=dtype)
                v = t.empty_like(k)
        self._run(self._lib.qnt_kv_read, self._p, layer, seqs.data_ptr(), first.data_ptr(), starts.data_ptr(), n, n_tok, k.data_ptr(),
                  v.data_ptr(), self._types[dtype], self._stream(stream))
        return k, v

    def attention(self, layer: int, q, seqs, starts, max_q: int, max_len: int, scale: float | None = None, window: int = 0,
                  lse: bool = False, stream=None):
        """Attention of q [tokens, n_heads, head_dim] over the cache of their sequences; query i of a sequence's m sits at
        position lens - m + i and sees the positions up to its own (the last `window` of them, if window > 0).  max_q bounds
        a sequence's queries, max_len its length.  Returns out (q's type), or (out, lse) with lse float32 [tokens, n_heads]."""
        dt, stride = self._rows("q", q)
        n_tok, heads = q.shape[:2]
        n = self._list(seqs, starts)
        if starts.numel() != n + 1:
            raise ValueError("starts must have one entry more than seqs")
        key = (heads, n, n_tok, max_q, max_len)
        need = self._need.get(key)
        if need is None:
            if len(self._need) > 4096:
                self._need.clear()
            need = self._need[key] = self._lib.qnt_kv_attention_workspace(self._p, heads, n, n_tok, max_q, max_len)
        s = self._stream(stream)
        w, nb = self._workspace(s, need)
        if stream is None:
            out = self._torch.empty_like(q)  # (a token's heads are contiguous and tokens do not overlap: so is this)
            ls = self.scales.new_empty((n_tok, heads)) if lse else None
        else:
            with self._allocating_on(stream):
                out = self._torch.empty_like(q)
                ls = self.scales.new_empty((n_tok, heads)) if lse else None
        self._run(self._lib.qnt_kv_attention, self._p, layer, q.data_ptr(), dt, stride, heads, seqs.data_ptr(), starts.data_ptr(), n,
                  n_tok, max_q, max_len, self.head_dim ** -0.5 if scale is None else scale, window,
                  out.data_ptr(), None if ls is None else ls.data_ptr(), w, nb, s)
        return (out, ls) if lse else out

    def check(self, stream=None):
        """Waits for the stream and raises the error that earlier calls on this cache ran into, if any."""
        self._run(self._lib.qnt_kv_check, self._p, self._stream(stream))


_torch_module = None


def _torch_calls():
    """quanta_b200_torch.so: the operators on torch tensors (csrc/torch_calls.cpp), of the folder that libquanta_b200.so is taken from."""
    global _torch_module
    if _torch_module is None:
        import importlib.machinery
        import importlib.util

        import torch  # noqa: F401  (its libraries come first)
        lib()
        p = LIB_DIR / "quanta_b200_torch.so"
        if not p.exists():
            raise RuntimeError(f"{p} is missing: run `python quanta.cpp_b200/build.py` where a torch with CUDA is installed")
        loader = importlib.machinery.ExtensionFileLoader("quanta_b200_torch", str(p))
        module = importlib.util.module_from_spec(importlib.util.spec_from_loader("quanta_b200_torch", loader))
        loader.exec_module(module)
        _torch_module = module
    return _torch_module


def _on_stream(stream, device):
    """torch.cuda.stream(stream) of a torch stream or a cudaStream_t's number."""
    from torch import cuda
    if not hasattr(stream, "cuda_stream"):
        stream = cuda.ExternalStream(int(stream), device=device) if int(stream) else cuda.default_stream(device)
    return cuda.stream(stream)


def rms_norm_q8(x, weight, eps: float = 1e-6, residual=None, stream=None):
    """RMS norm of rows x [tokens, n] (float32, float16 or bfloat16 CUDA tensor; rows may lie in wider ones) with 8-bit rows out:
    (q int8 [tokens, n], d float32 [tokens, n / 32]), the operand of the quantized products.  weight float32 [n].  With residual
    [tokens, n] (x's type or float32; the two must not overlap), residual += x first, in place, and the sum (before its rounding) is
    normed.  There are no gradients: results are outside autograd's graph, as within torch.no_grad(), and a tensor that a call writes
    in place is refused while a gradient is recorded through it.
    Work is queued on `stream` (a torch stream or a cudaStream_t's number; default: torch's current stream); with another one than
    the current one the call is as if made within torch.cuda.stream(stream).  So for the functions and objects below."""
    if stream is not None:
        with _on_stream(stream, x.device):
            return rms_norm_q8(x, weight, eps, residual)
    r = (_torch_module or _torch_calls()).rms_norm_q8(x, weight, eps, residual)
    return r if r.__class__ is tuple else _check(r)


_values = {}  # torch dtype -> number


def dequantize_q8(q, d, dtype=None, stream=None):
    """The values q * d of 8-bit rows (q int8 [tokens, n], d float32 [tokens, n / 32], contiguous CUDA tensors), as dtype (bfloat16
    unless said otherwise)."""
    if stream is not None:
        with _on_stream(stream, q.device):
            return dequantize_q8(q, d, dtype)
    if not _values:
        import torch
        _values.update({None: BF16, torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
    number = _values.get(dtype)
    if number is None:
        raise TypeError("dtype must be float32, float16 or bfloat16")
    r = (_torch_module or _torch_calls()).dequantize_q8(q, d, number)
    return _check(r) if r.__class__ is int else r


class Rope:
    """Rotary positions: rope(q, k, positions) rotates the first rotary_dim dims of every head (pairs (i, i + rotary_dim / 2), or with
    interleaved=True (2 i, 2 i + 1)) by positions * base ** (-2 i / rotary_dim); the other dims are copied.  scaling, for long contexts:
        dict(kind="linear", factor=)            every frequency divided by the factor
        dict(kind="ntk", factor=)               base * factor ** (rotary_dim / (rotary_dim - 2))
        dict(kind="yarn", factor=, original=, beta_fast=32, beta_slow=1, attention=None)  pairs that turn more than beta_fast times
            within the original context keep their frequency, those below beta_slow have it divided, a ramp between them; rotated
            values are multiplied by `attention` (0.1 ln factor + 1)
        dict(kind="bands", factor=, original=, low=1, high=4)  kept from `high` turns within the original context, divided up to
            `low`, a ramp between them
    or frequencies= (rotary_dim / 2 radians a position) instead of base and scaling."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: dict | None = None, frequencies=None,
                 device="cuda"):
        import torch
        self.rotary_dim, self.interleaved = int(rotary_dim), bool(interleaved)
        if self.rotary_dim <= 0 or self.rotary_dim % 2:
            raise ValueError("rotary_dim must be positive and even")
        if frequencies is None:
            f, self.scale = self.frequencies(self.rotary_dim, base, scaling)
        else:
            f, self.scale = [float(x) for x in frequencies], 1.0
            if len(f) != self.rotary_dim // 2 or scaling is not None:
                raise ValueError("frequencies: one for each pair, and no scaling beside them")
        self.turns = torch.tensor([x / (2 * math.pi) for x in f], dtype=torch.float64, device=device)  # revolutions a position
        self._inter = int(self.interleaved)

    @staticmethod
    def frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None):
        """(radians a position of each pair, factor on rotated values) of a base and a scaling, in 64 bits."""
        sc = dict(scaling or {"kind": "none"})
        kind = sc.pop("kind", None)
        known = {"none": {}, "linear": {"factor": None}, "ntk": {"factor": None},
                 "yarn": {"factor": None, "original": None, "beta_fast": 32.0, "beta_slow": 1.0, "attention": 0.0},
                 "bands": {"factor": None, "original": None, "low": 1.0, "high": 4.0}}
        if kind not in known or set(sc) - set(known[kind]):
            raise ValueError(f"scaling: kind none, linear, ntk, yarn or bands with {known.get(kind, {})}, not {scaling}")
        sc = known[kind] | {k: v for k, v in sc.items() if v is not None}
        if any(v is None for v in sc.values()) or any(v <= 0 for k, v in sc.items() if k in ("factor", "original", "beta_fast", "beta_slow")):
            raise ValueError(f"scaling {kind}: needs positive {[k for k in sc if known[kind][k] is None]}")
        if not base > 1:
            raise ValueError("base must be above 1")
        factor = sc.get("factor", 1.0)
        if kind == "ntk" and rotary_dim > 2:
            base = base * factor ** (rotary_dim / (rotary_dim - 2))
        f = [base ** (-2 * i / rotary_dim) for i in range(rotary_dim // 2)]
        if kind == "linear":
            return [x / factor for x in f], 1.0
        if kind == "yarn":
            lo, hi = (rotary_dim * math.log(sc["original"] / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (sc["beta_fast"], sc["beta_slow"]))
            lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rotary_dim - 1)
            ramp = [min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001))) for i in range(rotary_dim // 2)]
            return [x * (1 - r) + x / factor * r for x, r in zip(f, ramp)], sc["attention"] or 0.1 * math.log(factor) + 1.0
        if kind == "bands":
            if not sc["high"] > sc["low"]:
                raise ValueError("scaling bands: high must be above low")
            keep = [min(1.0, max(0.0, (sc["original"] * x / (2 * math.pi) - sc["low"]) / (sc["high"] - sc["low"]))) for x in f]
            return [x * k + x / factor * (1 - k) for x, k in zip(f, keep)], 1.0
        return f, 1.0

    def __call__(self, q, k, positions, inplace: bool = False, stream=None):
        """q [tokens, heads, head_dim] and k [tokens, kv heads, head_dim] (or None) of one type, float32, float16 or bfloat16; heads
        contiguous within a token, so that they may lie in the rows of one projection's output; positions int32 [tokens].
        Returns rotated (q, k), new contiguous tensors, or with inplace=True the ones given, which must not overlap."""
        if stream is not None:
            with _on_stream(stream, q.device):
                return self(q, k, positions, inplace)
        r = (_torch_module or _torch_calls()).rope(q, k, positions, self.turns, self.rotary_dim, self._inter, self.scale, inplace)
        return r if r.__class__ is tuple else _check(r)


class BeamSelector:
    """The selection of a beam search's next step (qnt_beam_select): select(logits, scores, ended) -> (scores float32, tokens int32,
    parents int32), each [groups, k], best first: of every group's candidates scores[g, b] + log_softmax(logits[g, b])[t] the k best,
    equal ones by the lowest beam, then token.  An ended beam has one candidate, its own score with token end_id.  Forbidden tokens
    (logits of -inf) and beams without a finite score come last, with -inf.  With k = beams, PagedKV.reorder takes the parents as
    they are.  Workspaces are one per stream and live as long as the object: a graph that captured calls is replayed while the
    object exists, ordered against the calls on the stream that it was captured on."""

    def __init__(self, k: int, end_id: int = -1):
        self.k, self.end_id = int(k), int(end_id)
        self._ws, self._kept = {}, []
        self._raw_stream = None

    def _workspace(self, device, stream, shape):
        """The stream's workspace, large enough for logits of this shape: (tensor, shapes that it is known to be enough for)."""
        import torch
        need = lib().qnt_beam_workspace(*shape, self.k) if len(shape) == 3 else 0
        if need == 0 and len(shape) == 3 and shape[0] > 0:
            raise QntError(-1, lib().qnt_last_error().decode(errors="replace"))
        ws = self._ws.get((device, stream))
        if ws is None or ws[0].numel() < need:
            size = max(need, 1 << 20)
            if ws is not None:  # the old one stays: queued kernels and captured graphs still write to it
                self._kept.append(ws[0])
                size = max(size, 2 * ws[0].numel())
            ws = self._ws[device, stream] = torch.empty(size, dtype=torch.uint8, device=f"cuda:{device}"), ws[1] if ws else set()
        if len(ws[1]) > 4096:
            ws[1].clear()
        ws[1].add(shape)
        return ws

    def __call__(self, logits, scores, ended=None, stream=None):
        """logits [groups, beams, vocab] (float32, float16 or bfloat16 CUDA tensor, rows at one distance, which may be wider than
        vocab), scores float32 [groups, beams], ended bool or uint8 [groups, beams] or None."""
        if stream is not None:
            with _on_stream(stream, logits.device):
                return self(logits, scores, ended)
        device, shape = logits.get_device(), logits.shape
        if device < 0:
            raise TypeError("logits must be a CUDA tensor")
        if self._raw_stream is None:
            import torch
            self._raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)
        s = self._raw_stream(device)
        ws = self._ws.get((device, s))
        if ws is None or shape not in ws[1]:
            ws = self._workspace(device, s, shape)
        r = (_torch_module or _torch_calls()).beam_select(logits, scores, ended, self.end_id, self.k, ws[0])
        return r if r.__class__ is tuple else _check(r)


def bench_mma_i8(iters: int = 4096) -> float:
    """Measured dense int8 tensor-core TOP/s of the current GPU (qnt_bench_mma_i8)."""
    v = C.c_double(0)
    _check(lib().qnt_bench_mma_i8(iters, C.byref(v)))
    return v.value

class Tokenizer:
    """Tokenizer (engine/src/tokenizer.h:15-39) of a .qnt file, on the host: encode(text) -> ids, decode(id) -> bytes,
    token_id(literal) -> special id or -1."""

    def __init__(self, path):
        h = C.c_void_p()
        _check(lib().qnt_tokenizer_open(str(path).encode(), C.byref(h)))
        self.h = h
        self.n_tokens = lib().qnt_tokenizer_n_tokens(h)

    def encode(self, text) -> np.ndarray:
        b = text.encode() if isinstance(text, str) else bytes(text)
        n = _check(lib().qnt_tokenize(self.h, b, len(b), None, 0))
        out = np.zeros(max(n, 1), np.int32)
        _check(lib().qnt_tokenize(self.h, b, len(b), _ptr(out), n))
        return out[:n]

    def decode(self, ids) -> bytes:
        if np.isscalar(ids):
            ids = [ids]
        parts = []
        for i in ids:
            n = _check(lib().qnt_token_piece(self.h, int(i), None, 0))
            buf = C.create_string_buffer(max(n, 1))
            lib().qnt_token_piece(self.h, int(i), buf, n)
            parts.append(buf.raw[:n])
        return b"".join(parts)

    def token_id(self, literal: str) -> int:
        return lib().qnt_token_id(self.h, literal.encode())

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.qnt_tokenizer_free(self.h)
        self.h = None

    __del__ = close

# ---------------------------------------------------------------- model level

def head_query(top_k=0, n_valid=0, must=None):
    must_arr = np.ascontiguousarray(must if must is not None else np.zeros(0), np.int32)
    hq = HeadQuery(top_k, n_valid, must_arr.ctypes.data_as(C.POINTER(C.c_int)), must_arr.size)
    hq._keep = must_arr
    return hq


class Model:
    """quanta::Model on the device (engine/src/model.h)."""

    def __init__(self, path: str | os.PathLike, ctx_len: int = 0, nibble_screen: bool = False):
        """nibble_screen: QNT_OPEN_NIBBLE_SCREEN (the shortlist head screens with the Q8 head's high nibble plane)."""
        h = C.c_void_p()
        _check(lib().qnt_model_open(str(path).encode(), ctx_len, 1 if nibble_screen else 0, C.byref(h)))
        self.h = h
        hp = HParams()
        _check(lib().qnt_model_hparams(h, C.byref(hp)))
        self.hp = hp
        self.vocab = hp.vocab_size
        self._logits = np.zeros(self.vocab, np.float32)

    def close(self):
        if getattr(self, "h", None) and _lib is not None:
            _lib.qnt_model_close(self.h)
        self.h = None

    __del__ = close

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    @staticmethod
    def _hq(hq):
        if hq is None:
            return None
        if isinstance(hq, HeadQuery):
            return C.byref(hq)
        return C.byref(head_query(**hq)) if isinstance(hq, dict) else hq

    def forward(self, token: int, pos: int, hq=None, copy: bool = True) -> np.ndarray | None:
        hqs = head_query(**hq) if isinstance(hq, dict) else hq
        _check(lib().qnt_model_forward(self.h, int(token), int(pos), C.byref(hqs) if hqs is not None else None,
                                       _ptr(self._logits) if copy else None))
        return self._logits.copy() if copy else None

    def forward_batch(self, tokens, pos0: int, hq=None, copy: bool = True) -> np.ndarray | None:
        t = np.ascontiguousarray(tokens, np.int32)
        hqs = head_query(**hq) if isinstance(hq, dict) else hq
        _check(lib().qnt_model_forward_batch(self.h, _ptr(t), t.size, int(pos0), C.byref(hqs) if hqs is not None else None,
                                             _ptr(self._logits) if copy else None))
        return self._logits.copy() if copy else None

    def head(self, hq=None, want_bounds: bool = False):
        hqs = head_query(**hq) if isinstance(hq, dict) else hq
        coarse = np.zeros(self.vocab, np.float32) if want_bounds else None
        upper = np.zeros(self.vocab, np.float32) if want_bounds else None
        _check(lib().qnt_model_head(self.h, C.byref(hqs) if hqs is not None else None, _ptr(self._logits), _ptr(coarse),
                                    _ptr(upper)))
        if want_bounds:
            return self._logits.copy(), coarse, upper
        return self._logits.copy()

    def nll(self, ids) -> float:
        """Sum over p of -log softmax(logits after ids[:p+1])[ids[p+1]] (the CLI's ppl); perplexity = exp(nll/(n-1))."""
        t = np.ascontiguousarray(ids, np.int32)
        v = C.c_double(0)
        _check(lib().qnt_model_nll(self.h, _ptr(t), t.size, C.byref(v)))
        return v.value

    @property
    def last_head_rows(self) -> int:
        return lib().qnt_model_last_head_rows(self.h)

    @property
    def has_shortlist(self) -> bool:
        return bool(lib().qnt_model_has_shortlist(self.h))

    @property
    def weight_bytes(self) -> int:
        return int(lib().qnt_model_weight_bytes(self.h))

    @property
    def packed_tensors(self) -> int:
        """Fused tensors this load took pre-packed from the file (export_device_layout); 0 for a plain .qnt."""
        return int(lib().qnt_model_packed_tensors(self.h))

    def generate(self, prompt, sp: SamplerParams, n_gen: int, shortlist: bool = True, batch_prefill: bool = True):
        """Session::feed + generate with the device sampler; returns (ids, stats dict)."""
        p = np.ascontiguousarray(prompt, np.int32)
        out = np.zeros(max(n_gen, 1), np.int32)
        spc = SamplerParamsC(sp.temperature, sp.top_k, sp.top_p, sp.min_p, sp.repeat_penalty, sp.repeat_window, sp.seed)
        st = GenStatsC()
        flags = (GEN_SHORTLIST if shortlist else 0) | (GEN_BATCH_PREFILL if batch_prefill else 0)
        n = _check(lib().qnt_generate(self.h, _ptr(p), p.size, C.byref(spc), flags, n_gen, _ptr(out), C.byref(st)))
        return out[:n].copy(), dict(prefill_ms=st.prefill_ms, decode_ms=st.decode_ms, head_rows=st.head_rows,
                                    head_calls=st.head_calls, kernels_per_step=st.kernels_per_step)


    # Session in pieces (qnt_session_begin / step / read)
    # ---- batched serving (greedy): many sequences with their own KV caches
    def batch_init(self, max_seqs: int, ctx_len: int):
        _check(lib().qnt_batch_init(self.h, max_seqs, ctx_len))

    def prefill_batch(self, seq: int, tokens) -> int:
        """Feeds the prompt of one sequence; returns its greedy next token."""
        t = np.ascontiguousarray(tokens, np.int32)
        nxt = C.c_int(-1)
        _check(lib().qnt_prefill_batch(self.h, seq, _ptr(t), t.size, C.byref(nxt)))
        return nxt.value

    def decode_batch(self, seq_ids, tokens) -> np.ndarray:
        """One greedy step of several distinct sequences; returns their next tokens."""
        s = np.ascontiguousarray(seq_ids, np.int32)
        t = np.ascontiguousarray(tokens, np.int32)
        out = np.empty(s.size, np.int32)
        _check(lib().qnt_decode_batch(self.h, _ptr(s), _ptr(t), s.size, _ptr(out)))
        return out

    def batch_reset(self, seq: int):
        _check(lib().qnt_batch_reset(self.h, seq))

    # the same with the paged 8-bit KV cache: prefill_batch, decode_batch and batch_reset as above
    def batch_init_paged(self, max_seqs: int, ctx_len: int, n_pages: int, page_tokens: int = 64):
        """Sequences take pages of page_tokens positions from one pool as they grow."""
        _check(lib().qnt_batch_init_paged(self.h, max_seqs, ctx_len, n_pages, page_tokens))

    def batch_fork(self, src: int, dst: int):
        """The empty sequence dst takes over src's positions (a shared prefix, another answer)."""
        _check(lib().qnt_batch_fork(self.h, src, dst))

    def batch_resize(self, n_pages: int):
        """Moves the pages in use into a pool of n_pages, which replaces the old one."""
        _check(lib().qnt_batch_resize(self.h, n_pages))

    def beam_search(self, prompt, beams: int, n_gen: int, end_id: int = -1):
        """Beam search from the paged cache (batch_init_paged first; sequences 0 .. beams - 1 must be empty and are so afterwards):
        (ids, score) of every beam, best first; ids end with end_id where the beam did."""
        t = np.asarray(prompt)
        for v in (beams, n_gen, end_id, *((t.min(), t.max()) if t.size else ())):
            if not -(2 ** 31) <= v < 2 ** 31:  # (a C int would take its lower half)
                raise ValueError(f"beam_search: {v} is past 32 bits")
        t = np.ascontiguousarray(t, np.int32)
        ids, lens, scores = np.zeros((max(beams, 1), max(n_gen, 1)), np.int32), np.zeros(max(beams, 1), np.int32), np.zeros(max(beams, 1), np.float32)
        _check(lib().qnt_beam_search(self.h, _ptr(t), t.size, beams, n_gen, end_id, _ptr(ids), _ptr(lens), _ptr(scores)))
        return [(ids[i, : lens[i]].copy(), float(scores[i])) for i in range(beams)]

    def session_begin(self, prompt, sp: SamplerParams, shortlist: bool = True, batch_prefill: bool = True):
        p = np.ascontiguousarray(prompt, np.int32)
        spc = SamplerParamsC(sp.temperature, sp.top_k, sp.top_p, sp.min_p, sp.repeat_penalty, sp.repeat_window, sp.seed)
        flags = (GEN_SHORTLIST if shortlist else 0) | (GEN_BATCH_PREFILL if batch_prefill else 0)
        _check(lib().qnt_session_begin(self.h, _ptr(p), p.size, C.byref(spc), flags))

    def session_step(self, n: int) -> int:
        return _check(lib().qnt_session_step(self.h, n))

    def session_feed(self, ids):
        t = np.ascontiguousarray(ids, np.int32)
        _check(lib().qnt_session_feed(self.h, _ptr(t), t.size))

    def session_rewind(self, n_drop: int):
        _check(lib().qnt_session_rewind(self.h, n_drop))

    def session_last(self):
        """(last sampled id, history length) after the queued steps."""
        tok, n = C.c_int(-1), C.c_int(0)
        _check(lib().qnt_session_last(self.h, C.byref(tok), C.byref(n)))
        return tok.value, n.value

    def session_read(self, max_ids: int = 1 << 16):
        out = np.zeros(max(max_ids, 1), np.int32)
        st = GenStatsC()
        n = _check(lib().qnt_session_read(self.h, _ptr(out), max_ids, C.byref(st)))
        return out[:n].copy(), dict(head_rows=st.head_rows, head_calls=st.head_calls, kernels_per_step=st.kernels_per_step)

    @property
    def stream(self) -> int:
        return int(lib().qnt_model_stream(self.h) or 0)


# ---------------------------------------------------------------- synthetic models

QWEN05B = dict(vocab_size=151936, dim=896, n_layers=24, n_heads=14, n_kv_heads=2, head_dim=64, ffn_dim=4864, max_seq=4096,
               rope_theta=1e6, norm_eps=1e-6, n_tokens=151665)
TINY = dict(vocab_size=5000, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=64, ffn_dim=512, max_seq=512,
            rope_theta=1e6, norm_eps=1e-6, n_tokens=4900)


def export_device_layout(src, dst) -> Path:
    """A copy of the .qnt at src, written to dst, with the device's fused q|k|v, gate|up and q|k|v-bias tensors stored
    pre-packed beside the original ones (which stay byte for byte, so the reference reads the copy unchanged).  No
    GPU needed."""
    _check(lib().qnt_export_device_layout(str(src).encode(), str(dst).encode()))
    return Path(dst)


def synth_model(path, *, shape: dict = QWEN05B, mlp_q4: bool = True, shortlist: bool = True, q4_group: int = 128,
                seed: int = 1234, w_std: float = 0.02, threads: int = 0, overwrite: bool = False, flags: int = 0,
                tokenizer: bytes | None = None) -> Path:
    """Writes a seeded random-init .qnt (q4mix = attention Q8_0 + MLP GPTQ-sym int4; or all Q8_0); flags = the header
    flags (1: FLAG_HADAMARD_DOWN); tokenizer = a complete tokenizer section (its token count must be shape's n_tokens)
    instead of the synthetic byte vocabulary."""
    global _synth
    path = Path(path)
    if path.exists() and not overwrite:
        return path
    if _synth is None:
        p = PKG / "lib" / "libqnt_synth.so"  # the model writer is not part of the phase-timed build
        if not p.exists():
            raise RuntimeError(f"{p} is missing: run `python quanta.cpp_b200/build.py`")
        _synth = C.CDLL(str(p))
        _synth.qnt_synth_write.argtypes = [C.c_char_p, C.POINTER(SynthCfg)]
        _synth.qnt_synth_last_error.restype = C.c_char_p
    cfg = SynthCfg(**{k: shape[k] for k in ("vocab_size", "dim", "n_layers", "n_heads", "n_kv_heads", "head_dim", "ffn_dim",
                                             "max_seq", "rope_theta", "norm_eps", "n_tokens")},
                   mlp_q4=int(mlp_q4), q4_group=q4_group, shortlist=int(shortlist), w_std=w_std, seed=seed,
                   n_threads=threads, flags=flags, tok_blob=tokenizer, tok_len=len(tokenizer) if tokenizer else 0)
    path.parent.mkdir(parents=True, exist_ok=True)
    tmp = path.with_suffix(path.suffix + f".tmp{os.getpid()}")
    if _synth.qnt_synth_write(str(tmp).encode(), C.byref(cfg)) != 0:
        raise RuntimeError(_synth.qnt_synth_last_error().decode())
    os.replace(tmp, path)
    return path
