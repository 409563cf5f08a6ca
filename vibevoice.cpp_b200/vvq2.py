"""ctypes binding of libvvq2.so (include/vvq2_capi.h) for tests, bench and
Python callers.  There is no fallback: if the shared library is missing or
no sm_100 device is present, calls raise."""
from __future__ import annotations

import ctypes as C
from pathlib import Path

import numpy as np

HERE = Path(__file__).resolve().parent
LIB_PATH = HERE / "libvvq2.so"

F32, F16, Q8_0, Q5_K, Q6_K, BF16 = 0, 1, 8, 13, 14, 30
ADVANCE, OUTPUT_NORM, LAST_ONLY = 1, 2, 4

LAYER_FIELDS = ["attn_norm", "attn_q", "attn_q_bias", "attn_k", "attn_k_bias", "attn_v",
                "attn_v_bias", "attn_o", "ffn_norm", "ffn_gate", "ffn_up", "ffn_down"]


class Tensor(C.Structure):
    _fields_ = [("data", C.c_void_p), ("type", C.c_int), ("ne0", C.c_int64), ("ne1", C.c_int64)]


class LayerWeights(C.Structure):
    _fields_ = [(n, Tensor) for n in LAYER_FIELDS]


class HParams(C.Structure):
    _fields_ = [("hidden_size", C.c_int), ("n_heads", C.c_int), ("n_kv_heads", C.c_int),
                ("head_dim", C.c_int), ("intermediate_size", C.c_int), ("n_layers", C.c_int),
                ("vocab_size", C.c_int), ("rope_theta", C.c_float), ("rms_norm_eps", C.c_float)]


class PagesDesc(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("block_table", C.c_void_p), ("n_layers", C.c_int),
                ("n_pages", C.c_int), ("max_pages", C.c_int), ("n_seqs", C.c_int), ("n_kv_heads", C.c_int),
                ("head_dim", C.c_int), ("type", C.c_int)]


class VVQ2Error(RuntimeError):
    def __init__(self, rc: int, msg: str):
        super().__init__(f"vvq2 error {rc}: {msg}")
        self.rc = rc


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise FileNotFoundError(f"{LIB_PATH} not built (run make -C vibevoice.cpp_b200)")
        L = C.CDLL(str(LIB_PATH))
        P, I, I64, F = C.c_void_p, C.c_int, C.c_int64, C.c_float
        sig = {
            "vvq2_init": (I, [P, I, P]),
            "vvq2_free": (None, [P]),
            "vvq2_set_layer": (I, [P, I, P]),
            "vvq2_set_output": (I, [P, P, P, P]),
            "vvq2_kv_init": (I, [P, I, I, P]),
            "vvq2_kv_init_paged": (I, [P, I, I, I, P]),
            "vvq2_kv_free_pages": (I, [P]),
            "vvq2_kv_free": (None, [P]),
            "vvq2_kv_load_prefix": (I, [P, I, I, P, P, I]),
            "vvq2_kv_read": (I, [P, I, I, P, P, I]),
            "vvq2_kv_set_past_len": (I, [P, I, I]),
            "vvq2_kv_past_len": (I, [P, I]),
            "vvq2_forward": (I, [P, P, P, I, I, P, P, I, I, I, P, P]),
            "vvq2_lm_head": (I, [P, I, P, P, P, P]),
            "vvq2_embed": (I, [P, I, P, P, P]),
            "vvq2_decode_step": (I, [P, P, P, I, P, P, P]),
            "vvq2_dequantize": (I, [I, P, I64, P]),
            "vvq2_rope_neox": (I, [P, I, I, I, P, F, P]),
            "vvq2_rms_norm": (I, [P, P, I, I, F, P]),
            "vvq2_backend_selected": (I, []),
            "vvq2_device_count": (I, []),
            "vvq2_version": (C.c_char_p, []),
            "vvq2_last_error": (C.c_char_p, []),
            "vvq2_kernel_launches": (I64, []),
            "vvq2_profile": (I, [P, I]),
            "vvq2_debug_gemm": (I, [I, P, I, I, P, I, P]),
            "vvq2_debug_gemv_mma": (I, [P, I, I, P, I, P]),
            "vvq2_attention_decode_noalloc": (I, [P, P, P, P, I, P, I, I, I, I, I, P, P, P]),
            "vvq2_attention_paged": (I, [P, I, P, I64, P, P, I, I, I, I, F, P, I64, P, P, C.c_size_t, P, P]),
            "vvq2_attention_paged_workspace": (C.c_size_t, [P, I, I, I, I]),
            "vvq2_attention_key_weights": (I, [P, I, P, I64, P, P, P, I, I, I, I, F, P, P, I64, P, C.c_size_t, P, P]),
            "vvq2_attention_key_weights_workspace": (C.c_size_t, [P, I, I, I, I]),
            "vvq2_pages_evict": (I, [P, P, I, P, I, P, I64, I, I, I, P, P, P, P, P]),
            "vvq2_profile_read": (I, [P, I, P, P, P]),
            "vvq2_mega_trace": (I, [P, P, C.c_int64, P, P]),
            "vvq2_nccl_unique_id": (I, [P]),
            "vvq2_partition": (I, [P, I, I, I, P]),
            "vvq2_set_connector": (I, [P, P, P, P, P, P]),
            "vvq2_connector": (I, [P, P, I, P, P]),
            "vvq2_set_eos": (I, [P, P, P, P, P]),
            "vvq2_eos": (I, [P, P, I, P, P]),
        }
        for name, (res, args) in sig.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def _chk(rc: int) -> int:
    if rc < 0:
        raise VVQ2Error(rc, lib().vvq2_last_error().decode())
    return rc


def _p(a) -> int | None:
    if a is None:
        return None
    if isinstance(a, int):
        return a
    if hasattr(a, "data_ptr"):          # torch tensor (device or host)
        return a.data_ptr()
    return a.ctypes.data


def launches() -> int:
    return lib().vvq2_kernel_launches()


class Engine:
    """One vvq2_ctx: hparams + device-resident weights."""

    def __init__(self, hp: dict, device: int = 0):
        self.hp = dict(hp)
        h = HParams(hp["hidden"], hp["n_heads"], hp["n_kv_heads"], hp["head_dim"], hp.get("ffn", 0),
                    hp["n_layers"], hp.get("vocab", 0), hp.get("rope_theta", 1.0e6),
                    hp.get("rms_eps", 1.0e-6))
        ptr = C.c_void_p()
        _chk(lib().vvq2_init(C.byref(h), device, C.byref(ptr)))
        self.ctx = ptr.value

    def close(self):
        if getattr(self, "ctx", None):
            lib().vvq2_free(self.ctx)
            self.ctx = None

    def __del__(self):
        self.close()

    @staticmethod
    def _tensor(spec) -> Tensor:
        if spec is None or spec[0] is None:
            return Tensor(None, 0, 0, 0)
        raw, qt, ne0, ne1 = spec
        raw = np.ascontiguousarray(raw)
        return Tensor(raw.ctypes.data, qt, ne0, ne1), raw

    def set_layer(self, li: int, tensors: dict) -> None:
        lw = LayerWeights()
        keep = []
        for n in LAYER_FIELDS:
            t = self._tensor(tensors.get(n))
            if isinstance(t, tuple):
                keep.append(t[1])
                t = t[0]
            setattr(lw, n, t)
        _chk(lib().vvq2_set_layer(self.ctx, li, C.byref(lw)))

    def set_output(self, output_norm=None, lm_head=None, tok_embd=None) -> None:
        ts, keep = [], []
        for spec in (output_norm, lm_head, tok_embd):
            t = self._tensor(spec)
            if isinstance(t, tuple):
                keep.append(t[1])
                t = t[0]
            ts.append(t)
        # a tied table: same array object for lm_head and tok_embd -> same pointer
        _chk(lib().vvq2_set_output(self.ctx, *[C.byref(t) if t.data else None for t in ts]))

    def _tensors(self, specs):
        ts, keep = [], []
        for spec in specs:
            t = self._tensor(spec)
            if isinstance(t, tuple):
                keep.append(t[1])
                t = t[0]
            ts.append(t)
        return [C.byref(t) if t.data else None for t in ts], keep

    def set_connector(self, fc1_w, fc1_b, norm_w, fc2_w, fc2_b) -> None:
        """SpeechConnector weights (src/vibevoice_tts.cpp:464-501)."""
        args, keep = self._tensors((fc1_w, fc1_b, norm_w, fc2_w, fc2_b))
        _chk(lib().vvq2_set_connector(self.ctx, *args))

    def connector(self, x, y=None, stream=None):
        """x [batch][latent] -> y [batch][hidden] = fc2(rms_norm(fc1 x + b1) * norm) + b2."""
        if not hasattr(x, "data_ptr"):
            x = np.ascontiguousarray(x, np.float32)
        batch = x.shape[0]
        if y is None:
            y = np.empty((batch, self.hp["hidden"]), np.float32)
        _chk(lib().vvq2_connector(self.ctx, _p(x), batch, _p(y), stream))
        return y

    def set_eos(self, fc1_w, fc1_b, fc2_w, fc2_b) -> None:
        """EOS classifier weights (src/vibevoice_tts.cpp:503-537)."""
        args, keep = self._tensors((fc1_w, fc1_b, fc2_w, fc2_b))
        _chk(lib().vvq2_set_eos(self.ctx, *args))

    def eos(self, x, p=None, stream=None):
        """x [batch][hidden] -> p [batch] = sigmoid(fc2(relu(fc1 x + b1)) + b2)."""
        if not hasattr(x, "data_ptr"):
            x = np.ascontiguousarray(x, np.float32)
        batch = x.shape[0]
        if p is None:
            p = np.empty(batch, np.float32)
        _chk(lib().vvq2_eos(self.ctx, _p(x), batch, _p(p), stream))
        return p

    def profile(self, enable: bool) -> None:
        _chk(lib().vvq2_profile(self.ctx, int(enable)))

    def profile_read(self, kind: int):
        ms, by, n = C.c_double(), C.c_double(), C.c_int64()
        _chk(lib().vvq2_profile_read(self.ctx, kind, C.byref(ms), C.byref(by), C.byref(n)))
        return ms.value, by.value, n.value

    def partition(self, rank: int, world: int, seq_parts: int, nccl_id: bytes) -> None:
        """Attention partition over `world` GPUs (one Engine per process and GPU):
        rank r holds KV-head group r // seq_parts and sequence part r % seq_parts.
        Call on every rank before set_layer / kv()."""
        buf = C.create_string_buffer(bytes(nccl_id), NCCL_ID_BYTES)
        _chk(lib().vvq2_partition(self.ctx, rank, world, seq_parts, C.cast(buf, C.c_void_p)))

    def mega_trace(self) -> np.ndarray:
        """[slots][grid] %globaltimer stamps of the last persistent decode step."""
        g, sl = C.c_int(), C.c_int()
        _chk(lib().vvq2_mega_trace(self.ctx, None, 0, C.byref(g), C.byref(sl)))
        out = np.zeros((sl.value, g.value), np.uint64)
        _chk(lib().vvq2_mega_trace(self.ctx, _p(out), out.size, None, None))
        return out

    def kv(self, n_seqs: int, max_seq: int, pool_pages: int = 0) -> "KV":
        """pool_pages > 0: a paged cache whose sequences share that many pages."""
        return KV(self, n_seqs, max_seq, pool_pages)

    def forward(self, kv: "KV", seqs, x, pos_start, first_layer=0, n_layers=None, flags=ADVANCE,
                y=None, stream=None):
        seqs = np.ascontiguousarray(seqs, np.int32)
        pos = np.ascontiguousarray(pos_start, np.int32)
        if n_layers is None:
            n_layers = self.hp["n_layers"] - first_layer
        if hasattr(x, "data_ptr"):
            n_tok = x.shape[1]
            xp = x
        else:
            x = np.ascontiguousarray(x, np.float32)
            n_tok = x.shape[1]
            xp = x
        if y is None:
            shape = (seqs.size, self.hp["hidden"]) if flags & LAST_ONLY else (seqs.size, n_tok, self.hp["hidden"])
            y = np.empty(shape, np.float32)
        _chk(lib().vvq2_forward(self.ctx, kv.kv, _p(seqs), seqs.size, n_tok, _p(xp), _p(pos),
                                first_layer, n_layers, flags, _p(y), stream))
        return y

    def lm_head(self, h, want_logits=False):
        h = np.ascontiguousarray(h, np.float32).reshape(-1, self.hp["hidden"])
        n = h.shape[0]
        am = np.empty(n, np.int32)
        lg = np.empty((n, self.hp["vocab"]), np.float32) if want_logits else None
        _chk(lib().vvq2_lm_head(self.ctx, n, _p(h), _p(lg), _p(am), None))
        return (am, lg) if want_logits else am

    def embed(self, tok) -> np.ndarray:
        tok = np.ascontiguousarray(tok, np.int32)
        out = np.empty((tok.size, self.hp["hidden"]), np.float32)
        _chk(lib().vvq2_embed(self.ctx, tok.size, _p(tok), _p(out), None))
        return out

    def decode_step(self, kv: "KV", seqs, tokens_in, tokens_out=None, stream=None):
        seqs = np.ascontiguousarray(seqs, np.int32)
        if not hasattr(tokens_in, "data_ptr"):
            tokens_in = np.ascontiguousarray(tokens_in, np.int32)
        if tokens_out is None:
            tokens_out = np.empty(seqs.size, np.int32)
        _chk(lib().vvq2_decode_step(self.ctx, kv.kv, _p(seqs), seqs.size, _p(tokens_in), _p(tokens_out),
                                    stream))
        return tokens_out


class KV:
    """vvq2_kv: f16 paged resident KV cache for n_seqs sequences (pool_pages >
    0: the sequences take pages from a shared pool as they grow)."""

    def __init__(self, eng: Engine, n_seqs: int, max_seq: int, pool_pages: int = 0):
        self.eng = eng
        ptr = C.c_void_p()
        if pool_pages > 0:
            _chk(lib().vvq2_kv_init_paged(eng.ctx, n_seqs, max_seq, pool_pages, C.byref(ptr)))
        else:
            _chk(lib().vvq2_kv_init(eng.ctx, n_seqs, max_seq, C.byref(ptr)))
        self.kv = ptr.value

    def free_pages(self) -> int:
        return lib().vvq2_kv_free_pages(self.kv)

    def close(self):
        if getattr(self, "kv", None):
            lib().vvq2_kv_free(self.kv)
            self.kv = None

    def __del__(self):
        self.close()

    def load_prefix(self, seq: int, layer: int, k, v) -> None:
        """k, v: f32 [n_pos][n_kv*hd], numpy (host) or torch (host or device)."""
        if not hasattr(k, "data_ptr"):
            k = np.ascontiguousarray(k, np.float32)
            v = np.ascontiguousarray(v, np.float32)
        _chk(lib().vvq2_kv_load_prefix(self.kv, seq, layer, _p(k), _p(v), k.shape[0]))

    def read(self, seq: int, layer: int, n_pos: int):
        w = self.eng.hp["n_kv_heads"] * self.eng.hp["head_dim"]
        k = np.empty((n_pos, w), np.float32)
        v = np.empty((n_pos, w), np.float32)
        _chk(lib().vvq2_kv_read(self.kv, seq, layer, _p(k), _p(v), n_pos))
        return k, v

    def set_past_len(self, seq: int, n: int) -> None:
        _chk(lib().vvq2_kv_set_past_len(self.kv, seq, n))

    def past_len(self, seq: int) -> int:
        return _chk(lib().vvq2_kv_past_len(self.kv, seq))


NCCL_ID_BYTES = 128


def nccl_unique_id() -> bytes:
    """A fresh NCCL unique id (make it on one rank, share it with the others)."""
    buf = C.create_string_buffer(NCCL_ID_BYTES)
    _chk(lib().vvq2_nccl_unique_id(C.cast(buf, C.c_void_p)))
    return buf.raw


def dequantize(qtype: int, raw: np.ndarray, n: int) -> np.ndarray:
    raw = np.ascontiguousarray(raw)
    out = np.empty(n, np.float32)
    _chk(lib().vvq2_dequantize(qtype, _p(raw), n, _p(out)))
    return out


def rope_neox(x: np.ndarray, pos: np.ndarray, theta: float) -> np.ndarray:
    """x f32 [n_tok][n_heads][hd], pos int32 [n_tok]."""
    x = np.ascontiguousarray(x, np.float32)
    pos = np.ascontiguousarray(pos, np.int32)
    y = np.empty_like(x)
    _chk(lib().vvq2_rope_neox(_p(x), x.shape[0], x.shape[1], x.shape[2], _p(pos), theta, _p(y)))
    return y


def rms_norm(x: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    x = np.ascontiguousarray(x, np.float32)
    w = np.ascontiguousarray(w, np.float32)
    y = np.empty_like(x)
    rows = x.size // x.shape[-1]
    _chk(lib().vvq2_rms_norm(_p(x), _p(w), rows, x.shape[-1], eps, _p(y)))
    return y


def debug_gemm(qtype: int, raw: np.ndarray, n: int, k: int, x: np.ndarray) -> np.ndarray:
    """y = x . W^T through the tcgen05 prefill GEMM (test hook)."""
    raw = np.ascontiguousarray(raw)
    x = np.ascontiguousarray(x, np.float32)
    y = np.empty((x.shape[0], n), np.float32)
    _chk(lib().vvq2_debug_gemm(qtype, _p(raw), n, k, _p(x), x.shape[0], _p(y)))
    return y


def debug_gemv_mma(raw: np.ndarray, n: int, k: int, x: np.ndarray) -> np.ndarray:
    """y = x . W^T (1-2 rows, Q8_0) through the tensor-core decode GEMV math (test hook)."""
    raw = np.ascontiguousarray(raw)
    x = np.ascontiguousarray(x, np.float32)
    y = np.empty((x.shape[0], n), np.float32)
    _chk(lib().vvq2_debug_gemv_mma(_p(raw), n, k, _p(x), x.shape[0], _p(y)))
    return y


# ---- operators over caller-owned K/V pages (torch tensors on one GPU) -------

def _arg(ok: bool, what: str) -> None:
    if not ok:
        raise VVQ2Error(-2, what)


def _current_stream(device) -> int:
    """torch's current cudaStream_t (its raw getter spares a call 2 us)."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw(device.index) if raw and device.index is not None else torch.cuda.current_stream(device).cuda_stream


class _On:
    """The stream a call runs on, and the allocator's stream for what it makes:
    torch's current stream of the tensors' device, or the given one (a torch
    stream or a cudaStream_t as an int)."""

    __slots__ = ("ptr", "ctx")

    def __init__(self, device, stream):
        if stream is None:
            self.ptr, self.ctx = _current_stream(device), None
        else:
            import torch
            s = stream if hasattr(stream, "cuda_stream") else torch.cuda.ExternalStream(stream, device=device)
            self.ptr, self.ctx = s.cuda_stream, torch.cuda.stream(s)

    def make(self, f, *args, **kw):
        """f(*args) with what it allocates belonging to this stream."""
        if self.ctx is None:
            return f(*args, **kw)
        with self.ctx:
            return f(*args, **kw)


class Pages:
    """Caller-owned K/V pages: k, v f16 or bf16 [n_pages][n_kv][64][hd], or with
    a leading layer axis; block_table int32 [n_seqs][max_pages].  Holds the
    tensors; their contents may change between calls."""

    def __init__(self, k, v, block_table):
        import torch
        _arg(k.dtype in (torch.float16, torch.bfloat16) and v.dtype == k.dtype, "K and V pages must be f16 or bf16")
        _arg(k.dim() in (4, 5) and k.shape == v.shape and k.shape[-2] == 64, "pages must be [..][n_kv][64][head_dim]")
        _arg(k.is_contiguous() and v.is_contiguous(), "pages must be contiguous")
        _arg(block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.is_contiguous(),
             "block_table must be contiguous int32 [n_seqs][max_pages]")
        _arg(k.device == v.device == block_table.device, "pages and block_table on different devices")
        self.k, self.v, self.block_table = k, v, block_table
        self.dtype, self.device, self.int32, self.float32 = k.dtype, k.device, torch.int32, torch.float32
        self.n_layers = k.shape[0] if k.dim() == 5 else 1
        self.n_pages, self.n_kv, _, self.head_dim = k.shape[-4:]
        self.n_seqs, self.max_pages = block_table.shape
        self._d = PagesDesc(k.data_ptr(), v.data_ptr(), block_table.data_ptr(), self.n_layers, self.n_pages,
                            self.max_pages, self.n_seqs, self.n_kv, self.head_dim,
                            F16 if k.dtype == torch.float16 else BF16)
        self._p = C.addressof(self._d)
        self._scratch = {}

    def _workspace(self, on, query, *sizes):
        """A call's scratch, of the size that its entry point asks for."""
        import torch
        n = self._scratch.get((query, sizes))
        if n is None:
            n = getattr(lib(), query)(self._p, *sizes)
            if len(self._scratch) >= 256:
                self._scratch.clear()
            self._scratch[query, sizes] = n
        return on.make(torch.empty, n, dtype=torch.uint8, device=self.device) if n else None

    def _done(self, rc: int) -> None:
        """Raises a failed call's error; the sizes kept so far may come from a
        query that failed with it (no scratch: the call's slow form)."""
        if rc:
            self._scratch.clear()
            _chk(rc)


def _words(x, shape, dtype, what: str) -> None:
    _arg(x.dtype is dtype and x.shape == shape and x.is_contiguous(), what)


def _heads(x, pages: Pages, what: str) -> int:
    """Elements between the token rows of [tokens][heads][head_dim] (a single
    row's own stride says nothing)."""
    n, h, hd = x.shape
    if x.is_contiguous():
        return h * hd
    _arg(n == 0 or (x.stride(2) == 1 and (h == 1 or x.stride(1) == hd)), what)
    return x.stride(0) if n > 1 else h * hd


def _rows(pages: Pages, q, q_start, kv_len):
    """Checks a packed chunk; returns (total_q, n_heads, row stride)."""
    _arg(q.dtype is pages.dtype and q.dim() == 3 and q.shape[2] == pages.head_dim,
         "q must be [total_q][n_heads][head_dim] of the pages' type")
    stride = _heads(q, pages, "the heads of a token must be contiguous")
    _words(q_start, (pages.n_seqs + 1,), pages.int32, "q_start must be int32 [n_seqs + 1]")
    _words(kv_len, (pages.n_seqs,), pages.int32, "kv_len must be int32 [n_seqs]")
    return q.shape[0], q.shape[1], stride


def _no_grad(*tensors) -> None:
    """The operators have no backward: a result that gradients should flow
    through would come out silently detached."""
    if any(x is not None and x.requires_grad for x in tensors):
        import torch
        _arg(not torch.is_grad_enabled(), "a tensor requires grad: detach it, or call under torch.no_grad()")


def _err(err):
    if err is None:
        return None
    import torch
    _arg(err.dtype == torch.int32 and err.numel() >= 1, "err must be int32")
    return err.data_ptr()


def attention_paged(q, pages: Pages, q_start, kv_len, max_q: int, max_kv: int, layer: int = 0, scale=None, out=None,
                    want_lse: bool = False, lse=None, err=None, stream=None):
    """Causal attention of packed new tokens over pages (vvq2_attention_paged).

    q [total_q][n_heads][hd]; sequence s has rows q_start[s]:q_start[s + 1] and
    kv_len[s] cached keys, its new tokens' own among them.  scale defaults to
    1 / sqrt(hd).  Returns out, or (out, lse) with want_lse or a given lse; rows
    past q_start[-1] keep what out and lse held.  out may be q itself."""
    import torch
    total, nq, stride = _rows(pages, q, q_start, kv_len)
    _no_grad(q, pages.k, pages.v, out, lse)
    on = _On(pages.device, stream)
    if out is None:
        out, out_stride = on.make(torch.empty_like, q, memory_format=torch.contiguous_format), nq * pages.head_dim
    else:
        _arg(out.shape == q.shape and out.dtype is q.dtype, "out must have q's shape and type")
        out_stride = _heads(out, pages, "out's heads of a token must be contiguous")
    if lse is not None:
        _words(lse, (total, nq), pages.float32, "lse must be contiguous f32 [total_q][n_heads]")
    elif want_lse:
        lse = on.make(q.new_empty, (total, nq), dtype=pages.float32)
    ws = pages._workspace(on, "vvq2_attention_paged_workspace", total, max_q, max_kv, nq)
    pages._done((_lib or lib()).vvq2_attention_paged(
        pages._p, layer, q.data_ptr(), stride, q_start.data_ptr(), kv_len.data_ptr(), total, max_q, max_kv, nq,
        scale if scale is not None else pages.head_dim ** -0.5, out.data_ptr(), out_stride,
        None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(),
        0 if ws is None else ws.numel(), _err(err), on.ptr))
    return out if lse is None else (out, lse)


def attention_key_weights(q, lse, pages: Pages, q_start, kv_len, max_q: int, max_kv: int, w_in=None, w_out=None,
                          layer: int = 0, scale=None, err=None, stream=None):
    """What each cached key received from a chunk's queries
    (vvq2_attention_key_weights), with attention_paged's lse for the same chunk.

    w_in, w_out f32 [n_seqs][n_kv][w_stride >= max_kv] (may be the same tensor);
    without w_out a zeroed one of width max_kv is made.  Older keys' w_in is
    added.  Returns w_out; words from kv_len[s] on keep what they held."""
    import torch
    total, nq, stride = _rows(pages, q, q_start, kv_len)
    _words(lse, (total, nq), pages.float32, "lse must be contiguous f32 [total_q][n_heads]")
    _no_grad(q, lse, pages.k, w_in, w_out)
    on = _On(pages.device, stream)
    if w_out is None:
        shape = (pages.n_seqs, pages.n_kv, max_kv) if w_in is None else w_in.shape
        w_out = on.make(torch.zeros, shape, dtype=pages.float32, device=pages.device)
    shape = (pages.n_seqs, pages.n_kv, w_out.shape[-1])
    _words(w_out, shape, pages.float32, "w_out must be contiguous f32 [n_seqs][n_kv][w_stride]")
    if w_in is not None:
        _words(w_in, shape, pages.float32, "w_in must be as w_out")
    ws = pages._workspace(on, "vvq2_attention_key_weights_workspace", total, max_q, max_kv, nq)
    pages._done((_lib or lib()).vvq2_attention_key_weights(
        pages._p, layer, q.data_ptr(), stride, lse.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), total,
        max_q, max_kv, nq, scale if scale is not None else pages.head_dim ** -0.5,
        None if w_in is None else w_in.data_ptr(), w_out.data_ptr(), w_out.shape[2],
        None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), _err(err), on.ptr))
    return w_out


def pages_evict(pages: Pages, dst_table, kv_len, w, keep: int, n_first: int = 0, n_recent: int = 0, max_kv=None,
                kept=None, w_out=None, new_len=None, err=None, stream=None):
    """Shortens every sequence to at most `keep` keys per layer and KV head
    (vvq2_pages_evict): the first n_first, the last n_recent, and of the others
    those of largest w [n_layers][n_seqs][n_kv][w_stride] (no layer axis needed
    for one layer).  K and V rows move to the pages of dst_table; continue with
    Pages(pages.k, pages.v, dst_table).  Returns (kept, new_len, w_out)."""
    import torch
    lead = (pages.n_layers, pages.n_seqs, pages.n_kv)
    _arg(dst_table.dim() == 2, "dst_table must be contiguous int32 [n_seqs][dst_max_pages]")
    _words(dst_table, (pages.n_seqs, dst_table.shape[1]), pages.int32,
           "dst_table must be contiguous int32 [n_seqs][dst_max_pages]")
    _words(kv_len, (pages.n_seqs,), pages.int32, "kv_len must be int32 [n_seqs]")
    width = w.shape[-1]
    if w.dim() == 3 and pages.n_layers == 1:
        lead = lead[1:]
    _words(w, (*lead, width), pages.float32, "w must be contiguous f32 [n_layers][n_seqs][n_kv][w_stride]")
    _arg(keep > 0, "keep must be positive")
    _no_grad(pages.k, pages.v, w, w_out)
    on, shape = _On(pages.device, stream), (*lead, keep)
    if kept is None:
        kept = on.make(torch.empty, shape, dtype=pages.int32, device=pages.device)
    if w_out is None:
        w_out = on.make(torch.empty, shape, dtype=pages.float32, device=pages.device)
    if new_len is None:
        new_len = on.make(torch.empty, pages.n_seqs, dtype=pages.int32, device=pages.device)
    _words(kept, shape, pages.int32, "kept must be contiguous int32 [n_layers][n_seqs][n_kv][keep]")
    _words(w_out, shape, pages.float32, "w_out must be contiguous f32, of kept's shape")
    _words(new_len, (pages.n_seqs,), pages.int32, "new_len must be int32 [n_seqs]")
    _chk((_lib or lib()).vvq2_pages_evict(pages._p, dst_table.data_ptr(), dst_table.shape[1], kv_len.data_ptr(),
                                          width if max_kv is None else max_kv, w.data_ptr(), width, keep, n_first,
                                          n_recent, kept.data_ptr(), w_out.data_ptr(), new_len.data_ptr(), _err(err),
                                          on.ptr))
    return kept, new_len, w_out
