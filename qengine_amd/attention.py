"""Attention over whole prompts and over a paged cache of keys and values, with the cache's own operations (the C-ABI's
qe_attn_* and qe_kv_* entry points, include/qe_kernels.h).

A serving step of a batch:

    cache = KVCache.empty(layers, pages, page, kv_heads, head_dim, slots, max_tokens)
    cache.reserve(seqs, counts)                       # pages for the new rows
    for layer in ...:
        cache.append(layer, k, v, seqs, cu)           # the new rows' keys and values
        o = attn_prompt(q, k, v, cu)                  # a prompt's first pass, or
        o = cache.attend(layer, q, seqs, cu, most)    # one token a sequence, or a drafted chain or tree (mask)
    cache.accept(seqs, counts)                        # the rows are the sequence's now (path: those of a tree that were kept)
    cache.fork(parents, children); cache.release(seqs)

Lengths, tables and batches (seqs, cu, counts: int32) stay on the device, so that steps need no host synchronization and
can be captured into graphs. Shapes, types, devices and strides are checked here (TypeError, ValueError) before the call;
values on the device are checked by the kernels, which skip what is out of range. Calls run on the current stream of the
tensors' device.
"""
import ctypes

import torch

from .qe import typed

F16 = 16
MAX_NODES = 64
MAX_BATCH = 1024
MAX_SEQS = 4096
MAX_ROWS = 1 << 30
HEAD_DIMS = (64, 128, 256)
_TYPES = (torch.bfloat16, torch.float16)
_FN = {}
_STRIDES = {}
_current = torch._C._cuda_getDevice
_stream_of = torch._C._cuda_getCurrentRawStream


def _run(at, name, sig, *args):
    """the call on the current stream of the tensors' device `at`, which need not be the current one"""
    if at < 0:
        raise ValueError("tensors are on a GPU")
    f = _FN.get(name)
    if f is None:
        f = _FN[name] = typed(name, sig)
    if at == _current():
        f(*args, _stream_of(at))
        return
    with torch.cuda.device(at):
        f(*args, _stream_of(at))


# Decode loops call these wrappers for every layer and token, so the checks below read few attributes: devices are compared
# as numbers (-1: CPU), and each tensor's stride is asked for once.
def _rows(name, t, dims, dtype, at):
    """a [.., d] tensor that the kernels can read: its type, place and strides"""
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {dtype}, got {t.dtype}")
    s = t.stride()
    if len(s) != dims:
        raise ValueError(f"{name} has {dims} dimensions, got shape {tuple(t.shape)}")
    if t.get_device() != at:
        raise ValueError(f"{name} is on another device than the other tensors: {t.device}")
    if s[-1] != 1 or (s[0] | s[1]) & 7 or (dims > 3 and any(x & 7 for x in s[2:-1])):
        if t.numel():
            raise ValueError(f"{name}: a row's values lie together and its other strides are multiples of 8, got {s}")
    if t.data_ptr() & 15:
        raise ValueError(f"{name} is 16-byte aligned")


def _ints(name, t, shape, at, dtype=torch.int32):
    if t.dtype is not dtype:
        raise TypeError(f"{name} is {dtype}, got {t.dtype}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} is contiguous of shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != at:
        raise ValueError(f"{name} is on another device than the other tensors: {t.device}")


def _starts(cu, at):
    shape = cu.shape
    if len(shape) != 1 or shape[0] < 1:
        raise ValueError(f"cu has one more entry than there are sequences, got shape {tuple(shape)}")
    if cu.dtype is not torch.int32 or not cu.is_contiguous() or cu.get_device() != at:
        _ints("cu", cu, shape, at)
    return shape[0] - 1


def _dtype_of(t):
    if t.dtype not in _TYPES:
        raise TypeError(f"values are bfloat16 or float16, got {t.dtype}")
    return t.dtype


def _check_out(out, q, dtype, at):
    _rows("out", out, 3, dtype, at)
    if out.shape != q.shape:
        raise ValueError(f"out has q's shape {tuple(q.shape)}, got {tuple(out.shape)}")
    s, (t, heads, d) = out.stride(), q.shape
    if s[0] < heads * s[1] or s[1] < d:  # not row after row of heads side by side
        (near, n), (far, m) = sorted(((s[0], t), (s[1], heads)))
        if n > 1 and near < d or m > 1 and far < (near * (n - 1) if n > 1 else 0) + d:
            raise ValueError(f"out's rows overlap: shape {tuple(q.shape)}, strides {s}")


def _check_scale(scale):
    if scale is not None and not 2.0 ** -126 <= scale <= 2.0 ** 126:
        raise ValueError(f"scale is positive and in the range of fp32, got {scale}")


def attn_prompt(q, k, v, cu, scale=None, out=None, lse=False):
    """Causal attention of packed prompts: q [t][heads][d], k and v [t][kv heads][d] (views into one QKV product do),
    sequence b the rows cu[b] .. cu[b + 1] - 1. -> out like q; with lse=True (out, lse [t][heads] fp32). Rows before cu[0]
    and from cu[-1] on are left as they were in a given `out` (and have no meaning in a new one), which is memory of its own,
    not part of q, k or v."""
    t, heads, kv, d, n, fresh = _prompt_shapes(q, k, v, cu, scale, out)
    if fresh:
        out = torch.empty(t, heads, d, dtype=q.dtype, device=q.device)
    sums = torch.empty(t, heads, dtype=torch.float32, device=q.device) if lse else None
    if t and n:
        qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
        kr, vr = (ks[0], vs[0]) if t > 1 else (0, 0)  # one row: its row stride may be anything
        _run(q.get_device(), "qe_attn_prompt", "pllpllpllpllppiiiiifip", q.data_ptr(), qs[0], qs[1], k.data_ptr(), kr, ks[1],
             v.data_ptr(), vr, vs[1], out.data_ptr(), os[0], os[1], sums.data_ptr() if lse else None, cu.data_ptr(), n, t,
             heads, kv, d, d ** -0.5 if scale is None else scale, F16 if q.dtype == torch.float16 else 0)
    return (out, sums) if lse else out


def _prompt_shapes(q, k, v, cu, scale, out):
    dtype, at = _dtype_of(q), q.get_device()
    _rows("q", q, 3, dtype, at)
    _rows("k", k, 3, dtype, at)
    _rows("v", v, 3, dtype, at)
    t, heads, d = q.shape
    ks, kv = k.shape, k.shape[1]
    if ks != v.shape or ks[0] != t or ks[2] != d or d not in HEAD_DIMS or kv == 0 or heads % kv or not heads or heads > 65535 \
            or t > MAX_ROWS:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: the same rows (at most {MAX_ROWS}), d of "
                         f"{HEAD_DIMS}, heads a multiple of the kv heads")
    if t > 1 and (k.stride(0) >= 1 << 24 or v.stride(0) >= 1 << 24):
        raise ValueError(f"rows of k and v are less than 2^24 elements apart, got {k.stride(0)} and {v.stride(0)}")
    n = _starts(cu, at)
    if n > MAX_SEQS:
        raise ValueError(f"at most {MAX_SEQS} sequences, got {n}")
    _check_scale(scale)
    if out is not None:
        _check_out(out, q, dtype, at)
    return t, heads, kv, d, n, out is None


class _CacheStruct(ctypes.Structure):
    """include/qe_kernels.h qe_kv_cache_t"""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("layer_stride", ctypes.c_int64),
                ("page_stride", ctypes.c_int64), ("head_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("table", ctypes.c_void_p), ("length", ctypes.c_void_p), ("held", ctypes.c_void_p), ("ref", ctypes.c_void_p)]
    _fields_ += [(x, ctypes.c_int32) for x in ("layers", "pages", "page", "kv_heads", "d", "slots", "width", "f16")]


class KVCache:
    """Paged keys and values of all layers and the state of its pages, around tensors that the caller may also look at:
    k, v [layers][pages][kv heads][page][d] (any strides that the kernels can read: a [.., page, kv heads, d] pool goes in
    as its transposed view), table [slots][width] (-1: none), length [slots], held [slots], ref [pages], int32."""

    def __init__(self, k, v, table, length, held, ref):
        self.device, self.dtype = k.device, _dtype_of(k)
        dtype, self._dev = self.dtype, k.get_device()
        device = self._dev
        _rows("k", k, 5, dtype, device)
        _rows("v", v, 5, dtype, device)
        if k.shape != v.shape or k.stride() != v.stride() or not k.numel():
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} have the same shape and strides")
        layers, pages, kv, page, d = k.shape
        if k.stride(3) >= 1 << 24:
            raise ValueError(f"tokens of a page are less than 2^24 elements apart, got {k.stride(3)}")
        if d not in HEAD_DIMS or pages >= 1 << 29 or page < 16 or page > 1024 or page & (page - 1) or kv > 1024 or layers > 65535:
            raise ValueError(f"pools [layers][pages][kv heads][page][d] with d of {HEAD_DIMS}, at most 65535 layers, 1024 kv heads and "
                             f"pages of 16 to 1024 tokens, a power of two: got {tuple(k.shape)}")
        if table.dim() != 2 or not table.numel() or table.shape[1] * page > 2 ** 30:
            raise ValueError(f"table is [slots][pages of a slot], got {tuple(table.shape)}")
        slots, width = table.shape
        _ints("table", table, table.shape, device)
        _ints("length", length, (slots,), device)
        _ints("held", held, (slots,), device)
        _ints("ref", ref, (pages,), device)
        self.k, self.v, self.table, self.length, self.held, self.ref = k, v, table, length, held, ref
        self.layers, self.pages, self.page, self.kv_heads, self.d, self.slots, self.width = layers, pages, page, kv, d, slots, width
        s = k.stride()
        self._c = _CacheStruct(k.data_ptr(), v.data_ptr(), s[0], s[1], s[2], s[3], table.data_ptr(), length.data_ptr(),
                               held.data_ptr(), ref.data_ptr(), layers, pages, page, kv, d, slots, width,
                               int(dtype == torch.float16))
        self._at = ctypes.addressof(self._c)
        self._scale = d ** -0.5
        self._units = -(-width * page // 32)  # what attend counts tokens in, at the least

    @staticmethod
    def empty(layers, pages, page, kv_heads, d, slots, max_tokens, dtype=torch.bfloat16, device="cuda"):
        """a cache that holds nothing, for slots of up to max_tokens tokens"""
        # zeros: a NaN behind a page's rows would not change results, but make the kernels look again at what they read
        k = torch.zeros(layers, pages, kv_heads, page, d, dtype=dtype, device=device)
        ints = dict(dtype=torch.int32, device=k.device)
        return KVCache(k, torch.zeros_like(k), torch.full((slots, -(-max_tokens // page)), -1, **ints),
                       torch.zeros(slots, **ints), torch.zeros(slots, **ints), torch.zeros(pages, **ints))

    def _batch(self, name, t, n=None):
        shape = t.shape
        if len(shape) != 1:
            raise ValueError(f"{name} has one dimension, got shape {tuple(shape)}")
        if n is None:
            n = shape[0]
        if t.dtype is not torch.int32 or shape[0] != n or not t.is_contiguous() or t.get_device() != self._dev:
            _ints(name, t, (n,), self._dev)
        return n

    def _few(self, n):
        if n > MAX_BATCH:
            raise ValueError(f"at most {MAX_BATCH} sequences a call, got {n}")

    def reserve(self, seqs, add):
        """Room for add[i] more tokens in slot seqs[i], entries in order; the last page is copied first where other slots hold
        it too. -> int32 [n], 1: done, 0: nothing changed (not enough pages, no room in the table, a bad or repeated slot)."""
        n = self._batch("seqs", seqs)
        self._batch("add", add, n)
        self._few(n)
        got = torch.empty(5 * n + 4, dtype=torch.int32, device=self.device)  # the list of copies, then the answers
        if n:
            _run(self._dev, "qe_kv_reserve", "pppippp", self._at, seqs.data_ptr(), add.data_ptr(), n,
                 got.data_ptr() + 16 * (n + 1), got.data_ptr())
        return got[4 * n + 4:]

    def fork(self, parents, children):
        """Slot children[i] shares the pages of parents[i]'s committed tokens. -> int32 [n], 1: done, 0: nothing changed (a bad
        slot, a child that is not empty or is repeated, or a parent that is one of the call's children). Drafted tokens that the
        parent has not committed stay its own: commit them before a fork, since rows do not move in a page that is shared."""
        n = self._batch("parents", parents)
        self._batch("children", children, n)
        self._few(n)
        ok = torch.empty(n, dtype=torch.int32, device=self.device)
        if n:
            _run(self._dev, "qe_kv_fork", "pppipp", self._at, parents.data_ptr(), children.data_ptr(), n, ok.data_ptr())
        return ok

    def release(self, seqs, lengths=None):
        """Slot seqs[i] keeps its first lengths[i] tokens (none without lengths) and gives its other pages back."""
        n = self._batch("seqs", seqs)
        if lengths is not None:
            self._batch("lengths", lengths, n)
        self._few(n)
        if n:
            _run(self._dev, "qe_kv_release", "pppip", self._at, seqs.data_ptr(), None if lengths is None else lengths.data_ptr(), n)

    def append(self, layer, k, v, seqs, cu):
        """New rows k, v [t][kv heads][d] of one layer, or [layers][t][kv heads][d] of all (layer None): rows cu[b] ..
        cu[b + 1] - 1 go behind the committed tokens of slot seqs[b], into pages reserved before (after a fork or a cut
        again: rows are not written into a page that other slots hold too). Slots are distinct. Rows without room are left
        out and nothing says so here: reserve's answer does."""
        one = layer is not None
        dims, shape = (3, k.shape) if one else (4, k.shape)
        _rows("k", k, dims, self.dtype, self._dev)
        _rows("v", v, dims, self.dtype, self._dev)
        if v.shape != shape or shape[-2] != self.kv_heads or shape[-1] != self.d or shape[-3] > MAX_ROWS \
                or not (one or shape[0] == self.layers):
            raise ValueError(f"k {tuple(shape)} and v {tuple(v.shape)} are at most {MAX_ROWS} rows of {self.kv_heads} kv heads of {self.d}"
                             + ("" if one else f", of {self.layers} layers"))
        if one and not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        n, t = _starts(cu, self._dev), shape[-3]
        self._batch("seqs", seqs, n)
        if t and n:
            ks, vs = k.stride(), v.stride()
            key = (ks[0], ks[-3], ks[-2], vs[0], vs[-3], vs[-2], one)
            strides = _STRIDES.get(key)  # the C arrays of the strides that have come up
            if strides is None:
                if len(_STRIDES) > 255:
                    _STRIDES.clear()
                c = (ctypes.c_int64 * 6)(0 if one else ks[0], ks[-3], ks[-2], 0 if one else vs[0], vs[-3], vs[-2])
                strides = _STRIDES[key] = (ctypes.addressof(c), c)
            _run(self._dev, "qe_kv_append", "piipppppiip", self._at, layer if one else 0, 1 if one else self.layers,
                 k.data_ptr(), v.data_ptr(), strides[0], seqs.data_ptr(), cu.data_ptr(), n, t)

    def accept(self, seqs, count, path=None, length=None):
        """count[i] drafted tokens of slot seqs[i] are committed: the first ones, or those of path int32 [n][at most 64], whose
        rows move together in all layers. The new lengths go to `length` [slots], or the cache's own. Slots are distinct. What
        counts is `count`, up to the slot's pages: also rows are committed that append left out, or that could not move, since
        their page is shared. So only slots whose reserve answered 1 are appended to and committed."""
        n = self._batch("seqs", seqs)
        self._batch("count", count, n)
        most = 0
        if path is not None:
            if path.dim() != 2 or path.shape[1] > MAX_NODES:
                raise ValueError(f"path is [sequences][at most {MAX_NODES}], got {tuple(path.shape)}")
            most = path.shape[1]
            _ints("path", path, (n, most), self._dev)
        if length is not None:
            _ints("length", length, (self.slots,), self._dev)
        if n > 65535:
            raise ValueError(f"at most 65535 sequences a call, got {n}")
        if n:  # (a path of no columns has no address, but is one)
            _run(self._dev, "qe_kv_accept", "ppppiipp", self._at, seqs.data_ptr(), count.data_ptr(),
                 None if path is None else path.data_ptr() or seqs.data_ptr(), most, n, None if length is None else length.data_ptr())

    def attend(self, layer, q, seqs, cu, most, mask=None, scale=None, out=None, lse=False):
        """Attention of drafted tokens, appended before: row cu[b] + i of q [t][heads][d] is drafted token i of slot seqs[b]; it
        sees the slot's committed tokens and the drafted tokens whose bit is set in mask[cu[b] + i] (int64 [t]), without a mask
        those up to itself. most (at most 64): the largest number of rows of a sequence. -> out like q; with lse=True (out,
        lse [t][heads] fp32). Rows of no sequence, or past `most`, are left as they were in a given `out`."""
        at, dtype = self._dev, self.dtype
        _rows("q", q, 3, dtype, at)
        t, heads, d = q.shape
        if d != self.d or heads == 0 or heads % self.kv_heads or heads > 65535 or t > MAX_ROWS:
            raise ValueError(f"q {tuple(q.shape)}: at most {MAX_ROWS} rows of heads of {self.d}, a multiple of the {self.kv_heads} kv heads")
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} of {self.layers}")
        if not 1 <= most <= MAX_NODES:
            raise ValueError(f"1 to {MAX_NODES} drafted tokens a sequence, got {most}")
        n = _starts(cu, at)
        self._batch("seqs", seqs, n)
        if n > MAX_SEQS:
            raise ValueError(f"at most {MAX_SEQS} sequences, got {n}")
        if mask is not None:
            _ints("mask", mask, (t,), at, torch.int64)
        if n * self.kv_heads * -(-most * (heads // self.kv_heads) // 128) * self._units > 1 << 30:
            raise ValueError(f"{n} sequences of {most} rows over tables of {self.width} pages: more than 2^30 units of work")
        _check_scale(scale)
        if out is None:
            out = torch.empty(t, heads, d, dtype=dtype, device=self.device)
        else:
            _check_out(out, q, dtype, at)
        sums = torch.empty(t, heads, dtype=torch.float32, device=self.device) if lse else None
        if t and n:
            qs, os = q.stride(), out.stride()
            _run(at, "qe_attn_tree", "pipllpllpppiiipifp", self._at, layer, q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1],
                 sums.data_ptr() if lse else None, seqs.data_ptr(), cu.data_ptr(), n, t, most,
                 None if mask is None else mask.data_ptr(), heads, self._scale if scale is None else scale)
        return (out, sums) if lse else out
