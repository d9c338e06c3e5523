"""A key-value cache in the pages of an array: what attention layers keep of their tokens, behind the page cache.

Keys and values that the page cache does not hold lie on the store and are fetched by the waves that want them, like any other element of an
array.  The reference has no counterpart; the C-ABI is bam_kv_* of include/bam_amd.h.
"""
import ctypes
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from .host import Array, BamError, PageCache, Range, _chk, _current, _stream, _wants_gradients, c_u64, c_vp

_TYPES = {torch.bfloat16: 0, torch.float16: 1}

# the structs of include/bam_amd.h, packed at once: a call takes 3 us less than with a ctypes argument for each field
_SEQS = "QQPPPqQ"
_READ = struct.Struct("@" + _SEQS)
_APPEND = struct.Struct("@" + _SEQS + "Pqq" * 3 + "PPPPPQIIfi")
_ATTEND = struct.Struct("@" + _SEQS + "PqqPPPQQQIIIf")
_REORDER = struct.Struct("@QQPPPqQPPPPPQ")


def _packed(layout, *fields):
    try:
        return layout.pack(*fields)
    except (struct.error, OverflowError) as e:
        raise BamError(f"KVCache: an argument is not a number that its field can hold ({e})") from None


class KVCache:
    """Blocks of `block_tokens` tokens in the pages of `array` from `first_page` on, two pages to a block and head.

    The calls below share how sequences are given, all on the device in int32: `lens[b]` counts the tokens of sequence b, the new ones among them;
    `table[b, i]` is the block of its tokens i * block_tokens and on; rows starts[b] .. starts[b+1]-1 of the packed inputs are its newest tokens
    (starts None: one new token each).  They are queued on the current stream.  A block number outside the cache is not read or written.  There are no gradients: tensors
    that require them are refused where gradients are being recorded, and those with a tangent (forward_ad).  The cache's device has to be the current one.

    stored: what the pages hold.  None: numbers of `dtype`.  torch.float8_e4m3fn: half as many bytes, each row (a token's keys of a head, or its values) as eight-bit numbers of
    four significant bits and a power of two; keys are normed and turned in 64 bits and rounded once, to that.  The powers of two are `scales`, a byte for each row in device memory
    (uint8 [n_blocks, n_heads, 2, block_tokens]: keys, values): given, or made here.  A cache that is opened again over pages that hold something needs the scales that go with them.
    """

    def __init__(self, array, n_heads, head_dim, dtype=torch.bfloat16, first_page=0, n_blocks=None, _owned=(), stored=None, scales=None):
        self.L = _lib.load()
        self.h = c_vp()
        self._owned = list(_owned)
        if dtype not in _TYPES:
            raise BamError("KVCache: dtype must be torch.bfloat16 or torch.float16")
        if n_blocks is None:
            raise BamError("KVCache: n_blocks must be given")
        if stored not in (None, dtype, torch.float8_e4m3fn):
            raise BamError("KVCache: stored must be None (numbers of dtype) or torch.float8_e4m3fn")
        eight = stored is torch.float8_e4m3fn
        if scales is not None and not eight:
            raise BamError("KVCache: scales go with stored=torch.float8_e4m3fn")
        self.array = array
        self._index = array.device
        self.device = torch.device("cuda", array.device)
        self.n_heads, self.head_dim, self.dtype, self.stored = n_heads, head_dim, dtype, torch.float8_e4m3fn if eight else dtype
        what = (ctypes.byref(self.h), array.h, first_page, n_blocks, n_heads, head_dim, _TYPES[dtype])
        if eight:
            if head_dim < 1 or n_blocks < 1 or n_heads < 1:
                raise BamError("KVCache: n_blocks, n_heads and head_dim must be at least 1")
            shape = (n_blocks, n_heads, 2, 1 << max(0, (array.ranges[0].cache.info()["page_size"] // head_dim).bit_length() - 1))
            if scales is None:
                scales = torch.zeros(shape, dtype=torch.uint8, device=self.device)
                # rows that are appended on another stream come after this
                torch.cuda.current_stream(self.device).synchronize()
            elif scales.shape != shape or scales.dtype is not torch.uint8 or scales.get_device() != self._index or not scales.is_contiguous():
                raise BamError(f"KVCache: scales must be contiguous {list(shape)} in uint8 on {self.device}")
            _chk(self.L.bam_kv_create_e4m3(*what, scales.data_ptr(), scales.numel()), "bam_kv_create_e4m3")
        else:
            _chk(self.L.bam_kv_create(*what), "bam_kv_create")
        self.scales, self._scales_on = scales, set()
        out = (c_u64 * 4)()
        _chk(self.L.bam_kv_info(self.h, out), "bam_kv_info")
        self.block_tokens, self.n_blocks, self.pages_per_block, self.page_size = list(out)
        self._bytes = {}

    # ---- checks: each property of a tensor is asked for once, they are what a small call takes on the host ----

    def _queue(self):
        """the current stream: kernels go to the device that is current, which has to be the one that the cache's memory is on"""
        if _current() != self._index:
            raise BamError(f"KVCache: the current device must be {self.device}: call under torch.cuda.device")
        stream = _stream()
        if self.scales is not None and stream.value not in self._scales_on:
            # a handle may go while its calls are queued: once told, torch's allocator gives the memory to nobody else before what this stream has by then is done
            self.scales.record_stream(torch.cuda.current_stream(self.device))
            self._scales_on.add(stream.value)
        return stream

    def _no_grad(self, t, what):
        if (t.requires_grad or forward_ad._current_level >= 0) and _wants_gradients(t):
            raise BamError(f"KVCache: {what} requires gradients or has a tangent, and there are none: detach it, or call under torch.no_grad()")

    def _rows(self, t, what, heads=None):
        """(rows, heads, row stride, head stride) of a tensor of rows"""
        shape = t.shape
        if len(shape) != 3 or t.dtype is not self.dtype or t.get_device() != self._index or shape[2] != self.head_dim or (heads is not None and shape[1] != heads):
            raise BamError(f"KVCache: {what} must be [rows, {'heads' if heads is None else heads}, {self.head_dim}] of {self.dtype} on {self.device}")
        row, head, one = t.stride()
        if one != 1:
            raise BamError(f"KVCache: the numbers of a row of {what} must be next to each other")
        self._no_grad(t, what)
        return shape[0], shape[1], row, head

    def _seqs(self, n_rows, lens, table, starts):
        shape, width = lens.shape, table.shape
        if len(shape) != 1 or lens.dtype is not torch.int32 or lens.get_device() != self._index or (shape[0] > 1 and lens.stride()[0] != 1):
            raise BamError(f"KVCache: lens must be a contiguous int32 tensor on {self.device}")
        n = shape[0]
        if len(width) != 2 or table.dtype is not torch.int32 or table.get_device() != self._index or width[0] != n:
            raise BamError(f"KVCache: table must be [{n}, blocks] in int32 on {self.device}")
        stride, one = table.stride()
        if one != 1 and width[1] > 1:
            raise BamError("KVCache: the blocks of a sequence must be next to each other in the table")
        if starts is None:
            if n != n_rows:
                raise BamError("KVCache: without starts every sequence has one new row")
            at = 0
        else:
            if starts.shape != (n + 1,) or starts.dtype is not torch.int32 or starts.get_device() != self._index or (n and starts.stride()[0] != 1):
                raise BamError(f"KVCache: starts must be {n + 1} contiguous int32 numbers on {self.device}")
            at = starts.data_ptr()
        return n_rows, n, at, lens.data_ptr(), table.data_ptr(), stride, width[1]

    def _weights(self, t, what):
        if t is None:
            return 0
        if t.dtype is not self.dtype or t.shape != (self.head_dim,) or t.stride()[0] != 1 or t.get_device() != self._index:
            raise BamError(f"KVCache: {what} must be {self.head_dim} contiguous numbers of {self.dtype} on {self.device}")
        self._no_grad(t, what)
        return t.data_ptr()

    def _out(self, out, like):
        if out is None:
            return torch.empty(like.shape, dtype=self.dtype, device=self.device)
        if out.shape != like.shape or out.dtype is not self.dtype or out.get_device() != self._index or not out.is_contiguous():
            raise BamError("KVCache: out must be like q, and contiguous")
        return out

    # ---- calls ----

    def append(self, k, v, lens, table, starts=None, q=None, q_norm=None, k_norm=None, eps=1e-6, cos=None, sin=None, rotary="half", out=None):
        """Put the new rows into the cache.  Keys, and queries if there are any, are normed per head (x * rsqrt(mean x^2 + eps) * weight) where a weight is
        given, and their first 2 * cos.shape[1] numbers are turned by the angles of their positions: pairs (i, i + half) with rotary="half",
        neighbours with "pairs"; cos and sin are [positions, half] in float32.  Returns the queries (None without)."""
        n, _, *k_strides = self._rows(k, "k", self.n_heads)
        v_rows, _, *v_strides = self._rows(v, "v", self.n_heads)
        if v_rows != n:
            raise BamError("KVCache: k and v must have the same rows")
        seqs = self._seqs(n, lens, table, starts)
        if q is not None:
            q_rows, q_heads, *q_strides = self._rows(q, "q")
            if q_rows != n or q_heads == 0:
                raise BamError("KVCache: q must have the rows of k and at least one head")
            out = self._out(out, q)
            q_args = (q.data_ptr(), *q_strides, out.data_ptr())
        elif q_norm is not None or out is not None:
            raise BamError("KVCache: q_norm and out go with q")
        else:
            q_heads, q_args = 0, (0, 0, 0, 0)
        if rotary != "half" and rotary != "pairs":
            raise BamError('KVCache: rotary must be "half" or "pairs"')
        angles, rot = (0, 0, 0), 0
        if cos is not None and sin is not None:
            shape = cos.shape
            for t in (cos, sin):
                if len(shape) != 2 or t.shape != shape or t.dtype is not torch.float32 or t.get_device() != self._index or not t.is_contiguous():
                    raise BamError(f"KVCache: cos and sin must be contiguous [positions, half] in float32 on {self.device}")
                self._no_grad(t, "cos or sin")
            angles, rot = (cos.data_ptr(), sin.data_ptr(), shape[0]), 2 * shape[1]
        elif cos is not None or sin is not None:
            raise BamError("KVCache: cos and sin go together")
        what = _packed(_APPEND, *seqs, k.data_ptr(), *k_strides, v.data_ptr(), *v_strides, *q_args, self._weights(q_norm, "q_norm"), self._weights(k_norm, "k_norm"),
                       *angles, q_heads, rot, eps, rotary == "pairs")
        _chk(self.L.bam_kv_append(self.h, what, self._queue()), "bam_kv_append")
        return out if q is not None else None

    def read(self, n_rows, lens, table, starts=None):
        """The newest rows as the cache has them: (keys, values), [n_rows, heads, head_dim] each."""
        if n_rows < 0:
            raise BamError("KVCache: n_rows must not be negative")
        seqs = self._seqs(n_rows, lens, table, starts)
        k = torch.empty(n_rows, self.n_heads, self.head_dim, dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        _chk(self.L.bam_kv_read(self.h, _packed(_READ, *seqs), k.data_ptr(), v.data_ptr(), self._queue()), "bam_kv_read")
        return k, v

    def attend(self, q, lens, table, starts=None, max_new=None, max_len=None, scale=None, window=0, sinks=0, out=None, return_lse=False):
        """Attention of the newest tokens (their rows in q) over what the cache holds of their sequences: the token at position p sees t <= p and, with
        a window, those with p - t < window or t < sinks.  scale: head_dim ** -0.5 unless given.  max_new: the most new rows a sequence has (all rows unless given; those beyond are left as they are);
        max_len: about the longest sequence (the table's width unless given); they decide how the work is shared out.  Rows of no sequence are left as they are.
        Returns the output, or with return_lse (output, logarithm of the sum of exponentials)."""
        n, hq, row, head = self._rows(q, "q")
        seqs = self._seqs(n, lens, table, starts)
        if hq == 0 or hq % self.n_heads:
            raise BamError(f"KVCache: the heads of q must be a multiple of {self.n_heads}")
        if not 0 <= window <= 0x7fffffff or not 0 <= sinks <= 0x7fffffff or (max_new is not None and max_new < 1) or (max_len is not None and not 1 <= max_len <= 0x7fffffff):
            raise BamError("KVCache: window and sinks must be 31-bit numbers, max_new and max_len at least 1, max_len a 31-bit number")
        out = self._out(out, q)
        lse = torch.empty(n, hq, dtype=torch.float32, device=self.device) if return_lse else None
        if n and seqs[1]:
            max_new = 1 if starts is None else min(n if max_new is None else max_new, n)
            max_len = seqs[6] * self.block_tokens if max_len is None else max_len
            key = (seqs[1], max_new, hq, max_len, window, sinks)
            need = self._bytes.get(key)
            if need is None:
                b = c_u64(0)
                _chk(self.L.bam_kv_attend_bytes(self.h, *key, ctypes.byref(b)), "bam_kv_attend_bytes")
                if len(self._bytes) > 4096:
                    self._bytes.clear()
                need = self._bytes[key] = b.value
            # from torch's allocator, which keeps it for this stream, or for the graph that is being captured
            work = torch.empty(need, dtype=torch.uint8, device=self.device)
            what = _packed(_ATTEND, *seqs, q.data_ptr(), row, head, out.data_ptr(), 0 if lse is None else lse.data_ptr(), work.data_ptr(), need, max_new, max_len,
                           hq, window, sinks, self.head_dim ** -0.5 if scale is None else scale)
            _chk(self.L.bam_kv_attend(self.h, what, self._queue()), "bam_kv_attend")
        return (out, lse) if return_lse else out

    def reorder(self, parents, lens, table, spare):
        """The sequences that go on behind a choice of beams: new sequence i continues old sequence parents[i] (int32, in any order, as often as it is named).  Returns (lens, table, spare) of the
        new ones.  Full blocks are shared; a last block that is not full (of one old sequence each) goes to the first of the parent's children, and each other one gets a copy of its tokens in block
        spare[i], a block of nobody else's (int32, one for each new sequence; -1, or one that the cache does not have: the child's last tokens are not there).  spare comes back with those blocks replaced:
        in the order of the children, by the last blocks, not full ones, of old sequences that nobody continues, and by -1 where there are no more.  A parent that is not there gives a sequence of no
        tokens.  In the new table, blocks without tokens are -1."""
        n = parents.shape[0] if len(parents.shape) == 1 else -1
        for t, what in ((parents, "parents"), (spare, "spare")):
            if t.shape != (n,) or t.dtype is not torch.int32 or t.get_device() != self._index or (n > 1 and t.stride()[0] != 1):
                raise BamError(f"KVCache: {what} must be contiguous int32, one number for each new sequence, on {self.device}")
        n_old = lens.shape[0] if len(lens.shape) == 1 else -1
        _, _, _, lens_at, table_at, stride, width = self._seqs(n_old, lens, table, None)
        new_lens, new_spare = torch.empty(2, n, dtype=torch.int32, device=self.device)
        new_table, work = torch.empty(n, width, dtype=torch.int32, device=self.device), torch.empty(n_old + n, dtype=torch.int32, device=self.device)
        if n:
            what = _REORDER.pack(n_old, n, parents.data_ptr(), lens_at, table_at, stride, width, spare.data_ptr(), new_lens.data_ptr(), new_table.data_ptr(), new_spare.data_ptr(),
                                 work.data_ptr(), 4 * (n_old + n))
            _chk(self.L.bam_kv_reorder(self.h, what, self._queue()), "bam_kv_reorder")
        return new_lens, new_table, new_spare

    def close(self):
        if self.h:
            self.L.bam_kv_destroy(self.h)
            self.h = c_vp()
        for x in self._owned:
            x.close()
        self._owned = []

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def make_kv_cache(ctrl, n_blocks, n_heads, head_dim, page_size=4096, cache_pages=None, dtype=torch.bfloat16, device=0, disk_offset_bytes=0, max_range=64, stored=None, scales=None):
    """Page cache + one range + array + key-value cache of n_blocks blocks, stored from byte disk_offset_bytes (page aligned).  cache_pages: slots of the page cache (all
    pages of the blocks unless given, and 64 at least).  stored, scales: what the pages hold (KVCache)."""
    if disk_offset_bytes < 0 or page_size <= 0 or disk_offset_bytes % page_size:
        raise BamError("make_kv_cache: disk_offset_bytes must be the beginning of a page")
    n_pages = 2 * n_blocks * n_heads
    made = []                # what there is so far, the last first
    try:
        made.insert(0, PageCache(page_size, max(64, n_pages if cache_pages is None else cache_pages), device, ctrl, max_range))
        elems = n_pages * page_size // 8
        made.insert(0, Range(0, elems, disk_offset_bytes // page_size, n_pages, 0, page_size, made[0], device))
        made.insert(0, Array(elems, disk_offset_bytes, [made[0]], device))
        return KVCache(made[0], n_heads, head_dim, dtype, 0, n_blocks, _owned=made, stored=stored, scales=scales)
    except BaseException:
        # not left to the collector: the error may be kept for longer than the controller lives
        for x in made:
            x.close()
        raise
