"""Serving operators on device buffers: 8-bit projections, a paged KV cache, attention over shared prefixes.

For decoding several hypotheses, languages or continuations of a clip at once; the reference decodes one greedy hypothesis
per clip and has no counterpart.  Buffers are device addresses (whole numbers) of the model's GPU, e.g. a torch tensor's
``data_ptr()``; nothing here allocates or computes.  ``stream`` is a hipStream_t address to enqueue on without waiting (it may be
under graph capture), or None for the model's own stream, which the call waits for.  A program that uses torch as well
imports torch first, so that both share one HIP runtime.
"""
import ctypes

from . import lib as _lib
from .lib import AttentionBatch

_DT = {"f32": _lib.F32, "bf16": _lib.BF16}


def _dtype(name):
    if name not in _DT:
        raise ValueError(f"dtype must be 'f32' or 'bf16', not {name!r}")
    return _DT[name]


class Int8Linear:
    """y = (q(x) . w^T) * s_x * s_w + bias with 8-bit weights [N][K] (row stride ldw bytes, a multiple of 16) and a scale per
    output channel; x is rounded to 8 bits per row inside the call."""

    def __init__(self, model, w, w_scales, N, K, ldw=None, bias=None):
        self._m, self._lib = model, model._lib
        self.w, self.w_scales, self.bias = w, w_scales, bias
        self.N, self.K = int(N), int(K)
        self.ldw = int(ldw) if ldw is not None else (self.K + 15) // 16 * 16

    def workspace_bytes(self, rows):
        n = int(self._lib.q3asr_i8_workspace(self._m._h, int(rows), self.N, self.K))
        if n < 0:
            raise ValueError("Int8Linear: sizes out of range")
        return n

    def __call__(self, x, rows, out, x_dtype="bf16", ldx=None, out_dtype="bf16", ldo=None, workspace=(None, 0), stream=None):
        """x [rows][ldx] -> out [rows][ldo]; workspace: (address, bytes)."""
        _lib.check(self._lib, self._lib.q3asr_i8_linear(
            self._m._h, x, _dtype(x_dtype), self.K if ldx is None else ldx, self.w, self.ldw, self.w_scales, self.bias, rows, self.N, self.K,
            out, _dtype(out_dtype), self.N if ldo is None else ldo, workspace[0], workspace[1], stream))

    def matmul(self, a, a_scales, rows, out, lda=None, out_dtype="bf16", ldo=None, stream=None):
        """The product alone, for activations that quantize_rows has rounded (K a multiple of 16)."""
        _lib.check(self._lib, self._lib.q3asr_i8_matmul(
            self._m._h, a, self.K if lda is None else lda, a_scales, self.w, self.ldw, self.w_scales, self.bias, rows, self.N, self.K, out,
            _dtype(out_dtype), self.N if ldo is None else ldo, stream))


def quantize_rows(model, x, rows, cols, q, scales, x_dtype="bf16", ldx=None, ldq=None, stream=None):
    """Rows of x to 8 bits with one fp32 scale each (a weight matrix [N][K]: one per output channel)."""
    _lib.check(model._lib, model._lib.q3asr_i8_quantize(model._h, x, _dtype(x_dtype), cols if ldx is None else ldx, rows, cols, q,
                                                        (cols + 15) // 16 * 16 if ldq is None else ldq, scales, stream))


class PagedKVCache:
    """A KV cache whose pages sequences share (``q3asr_kv_pages``): all arrays are the caller's."""

    OK, BAD_INDEX, DUPLICATE, NO_PAGES, TOO_LONG, BAD_BATCH = range(6)

    def __init__(self, model, k, v, layers, pages, kv_heads, head_dim, page_tokens, table, lens, refs, status, max_seqs, max_seq_pages):
        self._m, self._lib = model, model._lib
        self.c = _lib.Q3Pages(k=k, v=v, table=table, lens=lens, refs=refs, status=status, layers=layers, pages=pages, kv_heads=kv_heads,
                              head_dim=head_dim, page_tokens=page_tokens, max_seqs=max_seqs, max_seq_pages=max_seq_pages)
        self._c = ctypes.byref(self.c)

    def _check(self, rc):
        _lib.check(self._lib, rc)

    def workspace_bytes(self):
        """Bytes that fork, free, reserve and compact need."""
        n = int(self._lib.q3asr_pages_workspace(self._c))
        if n < 0:
            raise ValueError("PagedKVCache: sizes out of range")
        return n

    def set_workspace(self, address, nbytes):
        self.c.workspace, self.c.workspace_bytes = address, nbytes

    def reset(self, stream=None):
        self._check(self._lib.q3asr_pages_reset(self._m._h, self._c, stream))

    def fork(self, dst, src, n, stream=None):
        """Sequences dst[i] become what src[i] was (-1: empty), all at once."""
        self._check(self._lib.q3asr_pages_fork(self._m._h, self._c, dst, src, n, stream))

    def free(self, seqs, n, stream=None):
        self._check(self._lib.q3asr_pages_free(self._m._h, self._c, seqs, n, stream))

    def reserve(self, seqs, tokens, n, stream=None):
        """Room for tokens[i] more tokens of seqs[i]; a partly filled last page that others hold too is copied first."""
        self._check(self._lib.q3asr_pages_reserve(self._m._h, self._c, seqs, tokens, n, stream))

    def compact(self, stream=None):
        """The pages in use become the first ones of the pool."""
        self._check(self._lib.q3asr_pages_compact(self._m._h, self._c, stream))

    def status(self, clear=True, stream=None):
        """(code, entry, pages short of, pages in use after the last compact), after all that is enqueued on the stream."""
        out = (ctypes.c_int32 * 4)()
        self._check(self._lib.q3asr_pages_status(self._m._h, self._c, out, int(clear), stream))
        return tuple(out)

    def write(self, layer, k_rows, v_rows, batch, k_ld=None, v_ld=None, stream=None):
        """The step's K / V rows into the sequences' last positions."""
        width = self.c.kv_heads * self.c.head_dim
        self._check(self._lib.q3asr_pages_write(self._m._h, self._c, layer, k_rows, width if k_ld is None else k_ld, v_rows,
                                                width if v_ld is None else v_ld, batch, stream))

    def attention_workspace_bytes(self, batch, heads):
        n = int(self._lib.q3asr_paged_attention_workspace(self._m._h, self._c, batch, heads))
        if n < 0:
            raise _lib.Q3Error(self._lib.q3asr_last_error().decode("utf-8", "replace"))
        return n

    def attention(self, layer, q, out, batch, heads, scale=None, q_ld=None, o_ld=None, lse=None, workspace=(None, 0), stream=None):
        """Attention of the step's query rows over their sequences' keys (scale: head_dim ** -0.5 by default)."""
        d = self.c.head_dim
        self._check(self._lib.q3asr_paged_attention(
            self._m._h, self._c, layer, q, heads * d if q_ld is None else q_ld, heads, d ** -0.5 if scale is None else scale, batch, out,
            heads * d if o_ld is None else o_ld, lse, workspace[0], workspace[1], stream))
