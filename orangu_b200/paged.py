"""Operators over the pages of a cache that the caller holds (``ob_pages_*`` of the C ABI): attention of drafted trees, attention over chosen
pages, attention of new tokens over 4-bit pages or with the weights added up, what copies, forks and moves pages and positions and cuts caches
down; and the verification of drafted tokens (``ob_drafts_verify``).

Arrays are device arrays of the caller with ``data_ptr()``, ``shape``, ``dtype``, ``stride()`` and ``device``, as torch tensors have; this package
does not import torch.  Shapes and types are checked here, memory and ranges by the library.  Every call is asynchronous on ``stream``
(a ``cudaStream_t`` as a number, as ``torch.cuda.current_stream().cuda_stream`` gives it, 0 being the device's default stream; None is the
context's own stream, which is not ordered with any of those)."""
from __future__ import annotations

import ctypes as C

from . import capi
from .backend import CudaBackend

_PAGE = 16
_TYPES = {"float32": 0, "float16": capi.TYPE_F16, "bfloat16": capi.TYPE_BF16}


class _Kinds(dict):
    """dtype -> whether it is one of the named ones."""

    def __init__(self, *names):
        self.names = names

    def __missing__(self, dtype):
        ok = self[dtype] = str(dtype).replace("torch.", "") in self.names
        return ok


_INT, _INT32, _INT8, _WORDS, _FLOAT = _Kinds("int32", "uint32"), _Kinds("int32"), _Kinds("int8"), _Kinds("int64", "uint64"), _Kinds("float32")


def _stream(stream):
    return 1 if stream == 0 else stream  # to the C ABI null is the context's stream; 1 is what the runtime calls the legacy default stream


def _array(name, a, shape, kinds):
    """Address of a contiguous array of that shape."""
    if a.shape == shape and kinds[a.dtype] and a.is_contiguous():
        return a.data_ptr()
    if a.shape != shape:
        raise ValueError(f"{name} is {list(a.shape)}, expected {list(shape)}")
    if not kinds[a.dtype]:
        raise ValueError(f"{name} is {a.dtype}, expected {kinds.names[0]}")
    raise ValueError(f"{name} is not contiguous")


class _Types(dict):
    """dtype -> the library's type of it, or None."""

    def __missing__(self, dtype):
        t = self[dtype] = _TYPES.get(str(dtype).replace("torch.", ""))
        return t


_type_of = _Types()


class PagedCache:
    """``k``, ``v``: [layers, pages, kv heads, 16, head_dim] float16 or bfloat16, or (pages in 4 bits, written by ``store``) [layers, pages, kv heads,
    9 * head_dim] uint8; ``tables``: [sequences, pages each] int32.  The arrays stay the caller's; the handle keeps them alive.  Calls on one object
    share its workspace and have to be ordered on the device."""

    def __init__(self, backend: CudaBackend, k, v, tables):
        self._h = None
        self._type, name = k.dtype, str(k.dtype).replace("torch.", "")
        self._q4 = len(k.shape) == 4 and name == "uint8"
        if not self._q4 and (len(k.shape) != 5 or k.shape[3] != _PAGE):
            raise ValueError(f"k is {list(k.shape)}, expected [layers, pages, kv heads, {_PAGE}, head_dim]")
        types = {"float16": capi.TYPE_F16, "bfloat16": capi.TYPE_BF16}
        if self._q4:
            types = {"uint8": capi.TYPE_Q4_PAGES}
        if name not in types:
            raise ValueError(f"k is {k.dtype}, expected float16 or bfloat16")
        shape = tuple(k.shape)
        if self._q4 and shape[3] % 9:
            raise ValueError(f"k is {list(shape)}, expected [layers, pages, kv heads, 9 * head_dim]")
        if len(tables.shape) != 2:
            raise ValueError(f"tables is {list(tables.shape)}, expected [sequences, pages each]")
        self.backend, self._lib, self._arrays = backend, backend._lib, (k, v, tables)
        self._device = getattr(k, "device", None)
        self.n_layer, self.n_pages, self.n_head_kv = shape[:3]
        self.head_dim = shape[3] // 9 if self._q4 else shape[4]
        self.n_seq, self.table_stride = tuple(tables.shape)
        d = capi.PagesDesc(_array("k", k, shape, _Kinds(name)), _array("v", v, shape, _Kinds(name)), self.n_pages * self.n_head_kv * (9 if self._q4 else _PAGE) * self.head_dim, types[name],
                           self.n_layer, self.n_pages, self.n_head_kv, self.head_dim, self.n_seq, self.table_stride, _array("tables", tables, tuple(tables.shape), _INT32))
        h = C.c_void_p()
        capi.check(backend._h, self._lib.ob_pages_create(backend._h, C.byref(d), C.byref(h)))
        self._h = h

    def close(self):
        if self._h:
            self._lib.ob_pages_destroy(self._h)  # (after the backend's close(), too: the handle knows)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, rc):
        if rc:
            capi.check(self.backend._h, rc)

    def synchronize(self, stream=None):
        """Waits for ``stream``.  Raises OranguError if a wait inside a kernel of attention_tree or attention_tokens ran out since this was last asked: its
        output is not valid then."""
        self._check(self._lib.ob_pages_synchronize(self._h, _stream(stream)))

    def _rows(self, name, a, dtype=None):
        """Address, rows, heads and row stride of queries or outputs [rows, heads, head_dim], rows any multiple of eight entries apart."""
        shape = a.shape
        if len(shape) != 3 or shape[2] != self.head_dim or a.dtype != (dtype or self._type):
            raise ValueError(f"{name} is {list(shape)} of {a.dtype}, expected [rows, heads, {self.head_dim}] of {dtype or self._type}")
        rows, heads, dim = shape
        if a.is_contiguous():
            return a.data_ptr(), rows, heads, heads * dim
        stride = a.stride()
        if stride[2] != 1 or (heads > 1 and stride[1] != dim):
            raise ValueError(f"{name}: the heads of a row are not contiguous")
        return a.data_ptr(), rows, heads, stride[0] if rows > 1 else heads * dim

    def attention_tree(self, q, first_token, n_ctx, visible, scale: float, out, max_drafts: int, max_context: int, layer: int = 0, stream=None):
        """Attention of drafted tokens ``q`` [tokens, heads, head_dim] into ``out``: token i of sequence s (tokens first_token[s] .. first_token[s + 1] - 1) sees
        the sequence's n_ctx[s] positions and, at the positions after them, the drafted tokens whose bits are set in visible[i] (64 bits).  No
        sequence has more than ``max_drafts`` (at most 64); ``max_context`` is about the longest context."""
        qp, n, heads, q_stride = self._rows("q", q)
        op, on, oheads, o_stride = self._rows("out", out)
        n_seq = n_ctx.shape[0]
        if (on, oheads) != (n, heads):
            raise ValueError(f"out is {list(out.shape)}, expected {list(q.shape)}")
        self._check(self._lib.ob_pages_attention_tree(
            self._h, layer, n_seq, qp, q_stride, n, _array("first_token", first_token, (n_seq + 1,), _INT), _array("n_ctx", n_ctx, (n_seq,), _INT),
            _array("visible", visible, (n,), _WORDS), heads, max_drafts, max_context, scale, op, o_stride, _stream(stream)))

    def _bounds(self, codes, scales):
        pages = (self.n_pages, self.n_head_kv)
        return _array("codes", codes, pages + (2, self.head_dim), _INT8), _array("scales", scales, pages, _FLOAT)

    def bounds(self, first_pos, n_pos, codes, scales, max_new: int, layer: int = 0, stream=None):
        """8-bit bounds of the keys of the pages that hold positions first_pos[s] .. n_pos[s] - 1 (at most ``max_new`` a sequence): codes [pages, kv heads, 2,
        head_dim] int8 (largest, smallest) and their units, scales [pages, kv heads] float32."""
        n_seq = n_pos.shape[0]
        cp, sp = self._bounds(codes, scales)
        self._check(self._lib.ob_pages_bounds(self._h, layer, n_seq, _array("first_pos", first_pos, (n_seq,), _INT), _array("n_pos", n_pos, (n_seq,), _INT), max_new, cp, sp, _stream(stream)))

    def select(self, q, codes, scales, n_pos, selected, max_pos: int, keep_first: int = 0, keep_last: int = 0, row_seq=None, stream=None):
        """Per row and kv head the pages that ``q``'s row reads, into ``selected`` [rows, kv heads, n] int32: the first ``keep_first``, the last ``keep_last``, and
        those whose bounds promise the largest products; ascending, -1 behind the last.  Row r is of sequence row_seq[r] (None: r) and sees n_pos[r] positions."""
        qp, n, heads, q_stride = self._rows("q", q)
        cp, sp = self._bounds(codes, scales)
        n_select = selected.shape[-1]
        self._check(self._lib.ob_pages_select(
            self._h, cp, sp, n, qp, q_stride, _array("row_seq", row_seq, (n,), _INT) if row_seq is not None else None, _array("n_pos", n_pos, (n,), _INT), heads, max_pos,
            n_select, keep_first, keep_last, _array("selected", selected, (n, self.n_head_kv, n_select), _INT32), _stream(stream)))

    def attention(self, q, selected, n_pos, scale: float, out, row_seq=None, layer: int = 0, stream=None):
        """Attention of every row over the positions below n_pos[row] of the pages in ``selected`` (numbers within the row's sequence)."""
        qp, n, heads, q_stride = self._rows("q", q)
        op, on, oheads, o_stride = self._rows("out", out)
        if (on, oheads) != (n, heads):
            raise ValueError(f"out is {list(out.shape)}, expected {list(q.shape)}")
        n_select = selected.shape[-1]
        self._check(self._lib.ob_pages_attention(
            self._h, layer, n, qp, q_stride, _array("row_seq", row_seq, (n,), _INT) if row_seq is not None else None, _array("n_pos", n_pos, (n,), _INT), heads,
            _array("selected", selected, (n, self.n_head_kv, n_select), _INT32), n_select, scale, op, o_stride, _stream(stream)))

    def copy(self, src, dst, stream=None):
        """Page dst[i] of every layer becomes a copy of page src[i]; no page is written by one pair and in another."""
        n = src.shape[0]
        self._check(self._lib.ob_pages_copy(self._h, n, _array("src", src, (n,), _INT32), _array("dst", dst, (n,), _INT32), _stream(stream)))

    def fork(self, parent, child, n_pos, fresh, stream=None):
        """Sequence child[i] goes on from the first n_pos[i] positions of parent[i]: it shares the full pages; a last one that is not full is copied to page
        fresh[i]."""
        n = parent.shape[0]
        p = [_array(name, a, (n,), _INT) for name, a in (("parent", parent), ("child", child), ("n_pos", n_pos), ("fresh", fresh))]
        self._check(self._lib.ob_pages_fork(self._h, n, *p, _stream(stream)))

    def keep(self, n_ctx, kept, n_kept, stream=None, mass=None):
        """In all layers, position n_ctx[s] + kept[s, j] goes to n_ctx[s] + j for j < n_kept[s]: the accepted path of a tree of drafts moves together.  ``mass``
        [layers, sequences, kv heads, positions] float32 moves alike."""
        n_seq, width = kept.shape
        p = _array("n_ctx", n_ctx, (n_seq,), _INT), _array("kept", kept, (n_seq, width), _INT32), width, _array("n_kept", n_kept, (n_seq,), _INT)
        m = self._mass(mass, n_seq, self.n_layer) if mass is not None else None
        self._check(self._lib.ob_pages_keep(self._h, n_seq, *p, _stream(stream)))
        if m:
            self._check(self._lib.ob_pages_keep_mass(self._h, n_seq, *p, *m, _stream(stream)))

    def _mass(self, mass, n_seq, *layers):
        """Address and row stride of weights [(layers,) sequences, kv heads, positions], a table's positions or more."""
        width = mass.shape[-1]
        if width < self.table_stride * _PAGE:
            raise ValueError(f"mass is {list(mass.shape)}, expected at least {self.table_stride * _PAGE} positions")
        if getattr(mass, "device", None) != self._device:
            raise ValueError(f"mass is on {mass.device}, the cache on {self._device}")
        return _array("mass", mass, layers + (n_seq, self.n_head_kv, width), _FLOAT), width

    def _moved(self, call, k, v, first_token, n_ctx, max_tokens, layer, stream):
        t = _type_of[k.dtype]
        if not t:
            raise ValueError(f"k is {k.dtype}, expected float16 or bfloat16")
        kp, n, heads, k_stride = self._rows("k", k, k.dtype)
        vp, vn, vheads, v_stride = self._rows("v", v, k.dtype)
        if heads != self.n_head_kv or (vn, vheads) != (n, heads):
            raise ValueError(f"k is {list(k.shape)} and v {list(v.shape)}, expected [rows, {self.n_head_kv}, {self.head_dim}]")
        n_seq = n_ctx.shape[0]
        self._check(call(self._h, layer, n_seq, kp, vp, t, k_stride, v_stride, n, _array("first_token", first_token, (n_seq + 1,), _INT),
                         _array("n_ctx", n_ctx, (n_seq,), _INT), max_tokens, _stream(stream)))

    def store(self, k, v, first_token, n_ctx, max_tokens: int, layer: int = 0, stream=None):
        """4-bit pages: rows first_token[s] + j of ``k`` and ``v`` [tokens, kv heads, head_dim] (float16 or bfloat16) become positions n_ctx[s] + j of sequence
        s; no sequence has more than ``max_tokens``."""
        self._moved(self._lib.ob_pages_store, k, v, first_token, n_ctx, max_tokens, layer, stream)

    def load(self, k, v, first_token, n_ctx, max_tokens: int, layer: int = 0, stream=None):
        """4-bit pages: positions n_ctx[s] + j of sequence s become rows first_token[s] + j of ``k`` and ``v``; float16 holds them exactly."""
        self._moved(self._lib.ob_pages_load, k, v, first_token, n_ctx, max_tokens, layer, stream)

    def attention_tokens(self, q, first_token, n_ctx, scale: float, out, max_tokens: int, max_context: int, visible=None, mass=None, layer: int = 0, stream=None):
        """Attention of each sequence's newest tokens ``q`` [tokens, heads, head_dim] into ``out``, over pages of any type: token i of sequence s (tokens first_token[s] ..
        first_token[s + 1] - 1, at positions n_ctx[s], n_ctx[s] + 1, ...) sees the context, the tokens before it and itself, or, with ``visible``, the
        context and those of up to 64 tokens whose bits are set.  No sequence has more than ``max_tokens``; ``max_context`` is about the longest
        context.  ``mass`` [sequences, kv heads, positions] float32: the weights that positions get are added to those of the context, and
        those of the new positions are set to theirs."""
        dtype = q.dtype if self._q4 else self._type
        t = _type_of[dtype]
        if not t:
            raise ValueError(f"q is {q.dtype}, expected float16 or bfloat16")
        qp, n, heads, q_stride = self._rows("q", q, dtype)
        op, on, oheads, o_stride = self._rows("out", out, dtype)
        n_seq = n_ctx.shape[0]
        if (on, oheads) != (n, heads):
            raise ValueError(f"out is {list(out.shape)}, expected {list(q.shape)}")
        mp, m_stride = self._mass(mass, n_seq) if mass is not None else (None, 0)
        self._check(self._lib.ob_pages_attention_tokens(
            self._h, layer, n_seq, qp, t, q_stride, n, _array("first_token", first_token, (n_seq + 1,), _INT), _array("n_ctx", n_ctx, (n_seq,), _INT),
            _array("visible", visible, (n,), _WORDS) if visible is not None else None, heads, max_tokens, max_context, scale, op, o_stride, mp, m_stride, _stream(stream)))

    def evict(self, n_pos, mass, kept, n_left, max_pos: int, keep_first: int = 0, keep_last: int = 0, stream=None):
        """Cuts caches down, in all layers, to ``kept.shape[-1]`` positions: the first ``keep_first``, the last ``keep_last`` and those with the largest ``mass`` [layers,
        sequences, kv heads, positions]; keys, values and masses move together in order.  kept [layers, sequences, kv heads, n] int32: which positions they
        were, -1 behind the last; n_left[s] = min(n_pos[s], n).  ``max_pos`` is about the largest of n_pos."""
        n_seq, n = n_pos.shape[0], kept.shape[-1]
        mp, m_stride = self._mass(mass, n_seq, self.n_layer)
        self._check(self._lib.ob_pages_evict(
            self._h, n_seq, _array("n_pos", n_pos, (n_seq,), _INT), mp, m_stride, max_pos, n, keep_first, keep_last,
            _array("kept", kept, (self.n_layer, n_seq, self.n_head_kv, n), _INT32), _array("n_left", n_left, (n_seq,), _INT), _stream(stream)))


def verify_drafts(backend: CudaBackend, target, draft, tokens, parent, first_token, uniform, kept, n_kept, next_token, stream=None):
    """Which drafted tokens are accepted.  Node i of sequence s (nodes first_token[s] .. first_token[s + 1] - 1, node 0 the last certain token) is token tokens[i] and
    continues node parent[i] < i of its sequence; ``target`` [nodes, vocabulary] are the probabilities of what follows each node, ``draft`` those that its children were drawn
    from (None: each was certain), ``uniform`` [nodes] random numbers from [0, 1).  kept [sequences, up to 64] int32: node 0 and the accepted ones, no
    more than it has places, -1 behind them, as ``PagedCache.keep`` takes them; n_kept; next_token: what is drawn after the last of them."""
    t = _type_of[target.dtype]
    if t is None:
        raise ValueError(f"target is {target.dtype}, expected float32, float16 or bfloat16")
    n, vocab = target.shape
    n_seq = first_token.shape[0] - 1

    def rows(name, a):
        if tuple(a.shape) != (n, vocab) or a.dtype != target.dtype:
            raise ValueError(f"{name} is {list(a.shape)} of {a.dtype}, expected {[n, vocab]} of {target.dtype}")
        if vocab > 1 and a.stride()[1] != 1:
            raise ValueError(f"{name}: the probabilities of a row are not contiguous")
        return a.data_ptr(), a.stride()[0] if n > 1 else vocab

    tp, t_stride = rows("target", target)
    dp, d_stride = rows("draft", draft) if draft is not None else (None, 0)
    if len(kept.shape) != 2:
        raise ValueError(f"kept is {list(kept.shape)}, expected [sequences, up to 64]")
    rc = backend._lib.ob_drafts_verify(
        backend._h, n_seq, n, vocab, t, tp, t_stride, dp, d_stride, _array("tokens", tokens, (n,), _INT32), _array("parent", parent, (n,), _INT32),
        _array("first_token", first_token, (n_seq + 1,), _INT), _array("uniform", uniform, (n,), _FLOAT), _array("kept", kept, (n_seq, kept.shape[1]), _INT32), kept.shape[1],
        _array("n_kept", n_kept, (n_seq,), _INT), _array("next_token", next_token, (n_seq,), _INT32), _stream(stream))
    if rc:
        capi.check(backend._h, rc)
