"""A KV cache in pages, shared by many sequences, and the attention over it (l2_kv_* of include/llama2_b200.h) on torch CUDA tensors.

    pages = KvPages(k, v)                                   # [n_pages, page_size, kv_heads, head_size], f16 or bf16
    pages = KvPages(k, v, k_scale, v_scale)                 # int8, scales [n_pages, kv_heads, page_size] f32
    batch = KvBatch(page_table, kv_len, row_start, n_rows, max_rows)   # one step, for all layers
    pages.append(batch, k_rows, v_rows, rope=KvRope(4096), q=q_rows, q_out=q16)
    pages.attend(batch, q16, out, window=4096, sinks=4)
    pages.read(batch, k_back, v_back)

The objects keep the tensors they are made of.  Work is enqueued on the current torch stream unless `stream` (a cudaStream_t) is given; a call
does not wait for it.  With another stream than a tensor's own the caller orders the two and keeps rows and workspace until the work has run, as
with any torch kernel.  One host thread at a time uses a KvPages.
"""
import ctypes as C
import struct
import sys

from ._lib import KvBatchArgs, KvPagesArgs, KvRowsArgs, as_f32p, check, lib

F32, F16, BF16, I8, I32 = 0, 1, 2, 3, 4
BAD_PAGE, BAD_LENGTH, BAD_ROWS, BAD_ROPE, TIMEOUT = 1, 2, 4, 8, 16
_TYPES = {"torch.float32": F32, "torch.float16": F16, "torch.bfloat16": BF16, "torch.int8": I8, "torch.int32": I32}
_types = {}  # the same by dtype object, filled as they are seen
_ROWS2, _ROWS4 = struct.Struct("@" + "Pqqii" * 2), struct.Struct("@" + "Pqqii" * 4)  # l2_kv_rows, two and four in a row
_ROTATIONS = {"pairs": 0, "model": 1}  # L2_ROPE_*
_append, _read, _attend, _workspace_bytes = lib.l2_kv_append_rope, lib.l2_kv_read, lib.l2_kv_attend, lib.l2_kv_attend_workspace_bytes
assert _ROWS2.size == 2 * C.sizeof(KvRowsArgs) and _ROWS4.size == 4 * C.sizeof(KvRowsArgs)


def _type(t):
    d = t.dtype
    if d not in _types:
        _types[d] = _TYPES.get(str(d), -1)
    return _types[d]


_cuda = None  # torch's functions for the current device and its current stream, found at the first call without a stream


def _find_cuda():
    global _cuda
    torch = sys.modules["torch"]
    # (the raw stream without making a Stream object, which takes longer than the launch)
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
    _cuda = (getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device, raw)


def _stream(device, batch, stream):
    """The stream of a call, after a look at whether pages, batch and launch are all on one device."""
    if batch.device != device:
        raise ValueError("the batch is on device %d, the pages on device %d" % (batch.device, device))
    if _cuda is None:
        _find_cuda()
    if _cuda[0]() != device:
        raise ValueError("the tensors are on device %d, which is not the current one" % device)
    return _cuda[1](device) if stream is None else stream


def _packed(t, what, device, shape, dtype):
    if t.shape != shape or _type(t) != dtype or not t.is_contiguous() or t.get_device() != device:  # (-1: not on a CUDA device)
        raise ValueError("%s: contiguous %s of type code %d on device %d expected, got %s of %s" % (what, shape, dtype, device, tuple(t.shape), t.dtype))
    return t.data_ptr()


def _int32(**numbers):  # (ctypes would cut what is wider without a word)
    for what, n in numbers.items():
        if not -1 << 31 <= n < 1 << 31:
            raise ValueError("%s: %d is beyond 32 bits" % (what, n))


class KvBatch:
    """One step of a batch: page_table [n_seqs, width], kv_len [n_seqs] and row_start [n_seqs + 1] int32 on the device; n_rows rows in all,
    at most max_rows of one sequence.  `status` (one int32 on the device, optional) gets the BAD_* bits of what only the device can see."""

    def __init__(self, page_table, kv_len, row_start, n_rows, max_rows, status=None):
        if page_table.dim() != 2 or not page_table.is_cuda:
            raise ValueError("page_table: [n_seqs, width] on a CUDA device expected")
        self.device = page_table.get_device()
        n_seqs, width = page_table.shape
        _int32(n_seqs=n_seqs, table_width=width, n_rows=n_rows, max_rows=max_rows)
        self._args = KvBatchArgs(_packed(page_table, "page_table", self.device, (n_seqs, width), I32),
                                 _packed(kv_len, "kv_len", self.device, (n_seqs,), I32),
                                 _packed(row_start, "row_start", self.device, (n_seqs + 1,), I32),
                                 _packed(status, "status", self.device, (1,), I32) if status is not None else None,
                                 n_seqs, width, n_rows, max_rows)
        self._ref = C.byref(self._args)
        self._keep = (page_table, kv_len, row_start, status)
        self.n_rows = n_rows


class KvRope(tuple):
    """The tables of this package's models (l2_rope_table; heads of 128) for `positions` positions as two tensors on a device: (cos, sin).
    `append` turns with them as the models do, rotation "model"."""

    rotation = "model"

    def __new__(cls, positions, device="cuda"):
        import torch
        host = torch.empty((2, positions, 64))
        check(lib.l2_rope_table(positions, as_f32p(host[0].numpy()), as_f32p(host[1].numpy())))
        return super().__new__(cls, host.to(device))


class KvPages:
    """The pages of one layer's cache: k and v of one shape and one set of strides, [n_pages, page_size, kv_heads, head_size] (layout "NHD") or
    [n_pages, kv_heads, page_size, head_size] ("HND"), f16, bf16 or int8 (with scales)."""

    def __init__(self, k, v, k_scale=None, v_scale=None, layout="NHD"):
        if layout not in ("NHD", "HND"):
            raise ValueError("layout: NHD or HND")
        self.device = k.get_device()
        if k.dim() != 4 or self.device < 0 or v.get_device() != self.device:
            raise ValueError("k and v: four dimensions on a CUDA device expected")
        if v.shape != k.shape or v.dtype != k.dtype or v.stride() != k.stride() or k.stride(3) != 1:
            raise ValueError("k and v: the same shape, type and strides, the last dimension contiguous")
        at, head = (1, 2) if layout == "NHD" else (2, 1)
        self.n_pages, self.page_size, self.n_kv_heads, self.head_size = k.shape[0], k.shape[at], k.shape[head], k.shape[3]
        _int32(n_pages=self.n_pages, page_size=self.page_size, n_kv_heads=self.n_kv_heads)
        kind = _type(k)
        scales = [None, None]
        if kind == I8:
            if k_scale is None or v_scale is None:
                raise ValueError("an int8 cache needs k_scale and v_scale")
            shape = (self.n_pages, self.n_kv_heads, self.page_size)
            scales = [_packed(s, "scales", self.device, shape, F32) for s in (k_scale, v_scale)]
        elif k_scale is not None or v_scale is not None:
            raise ValueError("scales belong to an int8 cache")
        self._args = KvPagesArgs(k.data_ptr(), v.data_ptr(), scales[0], scales[1], k.stride(0), k.stride(at), k.stride(head), kind,
                                 self.n_pages, self.page_size, self.n_kv_heads, self.head_size)
        self._ref = C.byref(self._args)
        self._keep = (k, v, k_scale, v_scale)
        # the row records of a call, filled in place: making ctypes structures takes longer than the rest of it
        self._rows = (KvRowsArgs * 4)()
        self._at = tuple(C.addressof(self._rows) + i * C.sizeof(KvRowsArgs) for i in range(4))

    def _row(self, t, what, n, heads):
        """The fields of an l2_kv_rows for t; heads 0: as many as it has."""
        try:
            m, h, size = t.shape
            row, head, one = t.stride()
            kind = _types[t.dtype]
        except ValueError:
            m = h = size = one = -1
        except KeyError:
            kind = _type(t)
        if m != n or size != self.head_size or one != 1 or t.get_device() != self.device or (heads and h != heads):
            raise ValueError("%s: [%d, %s, %d] on device %d with its last dimension contiguous expected, got %s" % (what, n, heads or "heads", self.head_size, self.device, tuple(t.shape)))
        return t.data_ptr(), row, head, kind, h

    def append(self, batch, k, v, rope=None, q=None, q_out=None, stream=None, rotation=None):
        """K and V rows of the step into their pages; rope = (cos, sin), [positions, head_size / 2] f32, rotates k and, into q_out, q.
        rotation: "pairs" turns (x[d], x[d + head_size / 2]) as a vector; "model" does it in place, the second half from the turned first, as this
        package's models and l2_attention_decode_dev do (a cache of theirs, or their checkpoints).  Default: "model" for a KvRope, else "pairs"."""
        n, heads = batch.n_rows, self.n_kv_heads
        a = self._at
        if q is None and q_out is None:
            _ROWS2.pack_into(self._rows, 0, *self._row(k, "k", n, heads), *self._row(v, "v", n, heads))
            q_at = q_out_at = None
        else:
            if q is None or q_out is None:
                raise ValueError("q and q_out go together")
            _ROWS4.pack_into(self._rows, 0, *self._row(k, "k", n, heads), *self._row(v, "v", n, heads),
                             *self._row(q, "q", n, 0), *self._row(q_out, "q_out", n, q.shape[1]))
            q_at, q_out_at = a[2], a[3]
        cos = sin = None
        positions = turn = 0
        if rope is not None:
            cos, sin = rope
            turn = _ROTATIONS.get(rotation or getattr(rope, "rotation", "pairs"))
            if turn is None:
                raise ValueError("rotation: pairs or model")
            positions = cos.shape[0]
            shape = (positions, self.head_size // 2)
            cos, sin = _packed(cos, "rope", self.device, shape, F32), _packed(sin, "rope", self.device, shape, F32)
        rc = _append(self._ref, batch._ref, a[0], a[1], q_at, q_out_at, cos, sin, positions, turn, _stream(self.device, batch, stream))
        if rc:
            check(rc)

    def read(self, batch, k, v, stream=None):
        """The cached positions of the step's rows into k and v ([rows, kv_heads, head_size], f32, f16 or bf16)."""
        n, heads = batch.n_rows, self.n_kv_heads
        _ROWS2.pack_into(self._rows, 0, *self._row(k, "k", n, heads), *self._row(v, "v", n, heads))
        rc = _read(self._ref, batch._ref, self._at[0], self._at[1], _stream(self.device, batch, stream))
        if rc:
            check(rc)

    def workspace_bytes(self, batch, n_heads):
        _int32(n_heads=n_heads)
        n = _workspace_bytes(self._ref, batch._ref, n_heads)
        if not n:  # (never of a batch that is right)
            check(-1)
        return n

    def attend(self, batch, q, out, scale=None, window=0, sinks=0, workspace=None, stream=None):
        """Attention of the step's rows q [rows, heads, head_size] over the cache into out; scale defaults to head_size ** -0.5.
        `workspace`: a uint8 tensor of workspace_bytes(); one is made where none is given."""
        n = batch.n_rows
        if window >> 31 or sinks >> 31:
            _int32(window=window, sinks=sinks)
        row = self._row(q, "q", n, 0)
        _ROWS2.pack_into(self._rows, 0, *row, *self._row(out, "out", n, row[4]))
        if workspace is None:
            if stream is not None:
                raise ValueError("a stream of your own needs a workspace of your own: one made here is handed out again in the order of torch's stream")
            # (0 bytes of what is refused: the call says why)
            workspace = q.new_empty(_workspace_bytes(self._ref, batch._ref, row[4]), dtype=sys.modules["torch"].uint8)
        elif workspace.get_device() != self.device or not workspace.is_contiguous():
            raise ValueError("workspace: a contiguous tensor on the cache's device expected")
        rc = _attend(self._ref, batch._ref, self._at[0], self._at[1], self.head_size ** -0.5 if scale is None else scale, window, sinks,
                     workspace.data_ptr(), workspace.nbytes, _stream(self.device, batch, stream))
        if rc:
            check(rc)
        return out
