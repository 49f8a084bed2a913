"""The operators around an 8-bit key/value cache: kv_write, kv_read, KvAttention
and add_rms_norm over the C ABI (include/checkers_amd.h).

A KvCache names the cache's tensors, a KvBatch the tokens a call is about; both
are descriptors made once and passed to every call (the page table, starts and
offsets may change in place between calls: the kernels read them on the
device).  No call here copies or synchronises; only making a KvAttention does.

stream=: the stream a call's work is queued on, None: the current one.  As with
torch's own operators the caller orders it after the streams that made the
inputs, and keeps them (or records them on it) until it is done; outputs that
a call makes belong to that stream and may be used on the current one once that
waits for it.

None of this has a backward pass: tensors that require gradients are refused
where gradients are recorded (not under torch.no_grad()).
"""
import ctypes

from . import CKR_E_INVALID, BF16, F16, F32, I8, CkrError, _check, _torch, lib

F8 = 16  # 8-bit floating point (e4m3, largest value 448), a type of these operators only

_i64x3, _i64x2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2


class _Cache(ctypes.Structure):
    _fields_ = [("d_k", ctypes.c_void_p), ("d_v", ctypes.c_void_p), ("d_k_scale", ctypes.c_void_p),
                ("d_v_scale", ctypes.c_void_p), ("k_stride", _i64x3), ("v_stride", _i64x3),
                ("k_scale_stride", _i64x2), ("v_scale_stride", _i64x2), ("n_pages", ctypes.c_uint32),
                ("page_size", ctypes.c_uint32), ("n_heads", ctypes.c_uint32), ("head_dim", ctypes.c_uint32),
                ("dtype", ctypes.c_int32), ("pad", ctypes.c_int32)]


class _Batch(ctypes.Structure):
    _fields_ = [("d_page_table", ctypes.c_void_p), ("d_starts", ctypes.c_void_p), ("d_offsets", ctypes.c_void_p),
                ("table_stride", ctypes.c_uint64), ("table_width", ctypes.c_uint32), ("n_seqs", ctypes.c_uint32),
                ("n_tokens", ctypes.c_uint32), ("max_chunk", ctypes.c_uint32), ("max_context", ctypes.c_uint32),
                ("pad", ctypes.c_uint32)]


_TAGS = {}   # torch dtype -> tag


def _tag(dtype):
    """C tag of a torch dtype of these operators (8-bit floats among them)."""
    if not _TAGS:
        torch = _torch()
        _TAGS.update({torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16, torch.int8: I8,
                      torch.float8_e4m3fn: F8})
    tag = _TAGS.get(dtype)
    if tag is None:
        raise CkrError(CKR_E_INVALID, f"[ckr] {dtype} is not a type of the cache and norm operators")
    return tag


def _torch_dtype(tag):
    _tag(_torch().int8)
    for d, t in _TAGS.items():
        if t == tag:
            return d
    raise CkrError(CKR_E_INVALID, f"[ckr] tag {tag} is not a type of the cache and norm operators")


def _need(ok, msg):
    if not ok:
        raise CkrError(CKR_E_INVALID, "[ckr] " + msg)


def _on_gpu(t, what):
    _need(t.is_cuda, f"{what} must be on a GPU")


class KvCache:
    """A paged cache over the caller's tensors: k and v [pages, heads, page_size,
    head_dim] with any strides of the first three axes, for 8-bit types k_scale
    and v_scale [pages, heads, page_size] in float32 (slots contiguous)."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype, "k and v must be alike, [pages, heads, page_size, head_dim]")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "the last axis of k and v must be contiguous")
        self.dtype = _tag(k.dtype)
        coded = self.dtype in (F8, I8)
        _need(coded == (k_scale is not None) == (v_scale is not None), "scales belong to 8-bit caches, and to both k and v")
        for t, what in ((k, "k"), (v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if t is not None:
                _on_gpu(t, what)
                _need(t.device == k.device, "the cache's tensors must be on one GPU")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_heads, self.page_size, self.head_dim = k.shape
        c = _Cache(k.data_ptr(), v.data_ptr(), None, None, _i64x3(*k.stride()[:3]), _i64x3(*v.stride()[:3]),
                   _i64x2(0, 0), _i64x2(0, 0), *(int(n) for n in (k.shape[0], k.shape[2], k.shape[1], k.shape[3])),
                   self.dtype, 0)
        if coded:
            for t in (k_scale, v_scale):
                _need(t.shape == k.shape[:3] and t.dtype == _torch().float32 and t.stride(2) == 1,
                      "scales must be float32 [pages, heads, page_size], slots contiguous")
            c.d_k_scale, c.d_v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            c.k_scale_stride, c.v_scale_stride = _i64x2(*k_scale.stride()[:2]), _i64x2(*v_scale.stride()[:2])
        self._c = c
        self._p = ctypes.byref(c)

    @classmethod
    def empty(cls, n_pages, page_size, n_heads, head_dim, dtype, device="cuda"):
        """A cache of new tensors (dtype: F8, I8, BF16 or F16), zeroed."""
        torch = _torch()
        t = _torch_dtype(dtype)
        kv = [torch.zeros((n_pages, n_heads, page_size, head_dim), dtype=torch.uint8 if dtype == F8 else t, device=device)
              for _ in range(2)]
        if dtype == F8:
            kv = [x.view(t) for x in kv]
        sc = [torch.zeros((n_pages, n_heads, page_size), dtype=torch.float32, device=device) if dtype in (F8, I8) else None
              for _ in range(2)]
        return cls(kv[0], kv[1], sc[0], sc[1])

    def tensors(self):
        """The cache's tensors (k, v and, in 8 bits, their scales)."""
        return [t for t in (self.k, self.v, self.k_scale, self.v_scale) if t is not None]


class KvBatch:
    """The tokens of a call: sequence s has starts[s] tokens before its chunk,
    rows offsets[s]:offsets[s + 1] of the packed tensors, in the cache pages that
    page_table[s] lists (negative: unmapped; a table expanded from one row is read as
    such).  All int32 on the GPU; n_tokens is
    offsets[-1], max_chunk and max_context (the longest chunk, the largest
    context with its chunk) choose launches and need not be exact.  The longest
    chunk chooses for all sequences, so prompts and sequences that decode are
    faster in calls of their own."""

    def __init__(self, page_table, starts, offsets, n_tokens, max_chunk=None, max_context=None):
        torch = _torch()
        _need(page_table.dim() == 2 and (page_table.stride(1) == 1 or page_table.shape[1] == 1), "page_table must be [sequences, pages], its rows contiguous")
        n = page_table.shape[0]
        _need(tuple(starts.shape) == (n,) and tuple(offsets.shape) == (n + 1,), "starts and offsets must hold n and n + 1 entries")
        for t, what in ((page_table, "page_table"), (starts, "starts"), (offsets, "offsets")):
            _need(t.dtype == torch.int32 and (t.dim() == 2 or t.is_contiguous()), f"{what} must be int32, contiguous")
            _on_gpu(t, what)
        _need(0 <= n_tokens < 1 << 31, "n_tokens out of range")
        self.page_table, self.starts, self.offsets, self.n_seqs, self.n_tokens = page_table, starts, offsets, n, int(n_tokens)
        self.max_chunk = int(n_tokens if max_chunk is None else max_chunk)
        self.max_context = max_context
        width = page_table.shape[1]
        stride = page_table.stride(0) if n > 1 else width   # 0, or below the width: rows that share entries
        self._c = _Batch(page_table.data_ptr(), starts.data_ptr(), offsets.data_ptr(), stride,
                         width, n, self.n_tokens, min(self.max_chunk, 0xffffffff),
                         0xffffffff if max_context is None else min(int(max_context), 0xffffffff), 0)
        self._p = ctypes.byref(self._c)


def _stream_of(stream, tensor):
    """The stream's handle; None: the current stream of the tensor's GPU.  (A
    decoding step's calls last a few microseconds each, so neither this nor the
    checks below build objects that they do not need.)"""
    if stream is not None:
        return stream.cuda_stream
    return _torch()._C._cuda_getCurrentRawStream(tensor.get_device())


def _bad(msg):
    raise CkrError(CKR_E_INVALID, "[ckr] " + msg)


def _no_backward():
    """For inputs that require gradients: refused where one would be lost."""
    if _torch().is_grad_enabled():
        _bad("these operators have no backward pass: call them under torch.no_grad(), or on detached tensors")


def _rows(t, n_tokens, heads, dim, what):
    """(token stride, head stride) of a [tokens, heads, dim] tensor on a GPU."""
    shape = t.shape
    if len(shape) != 3 or shape[0] != n_tokens or shape[1] != heads or shape[2] != dim:
        _bad(f"{what} must be [{n_tokens}, {heads}, {dim}], not {list(shape)}")
    a, b, c = t.stride()
    if c != 1:
        _bad(f"the last axis of {what} must be contiguous")
    if not t.is_cuda:
        _bad(f"{what} must be on a GPU")
    return a, b


def _new(shape, dtype, device, stream):
    """An output of a call on `stream` (None: the current one).  Its memory is of that
    stream's, so whoever had it before has done with it there; the caller may go
    on with it on the current stream, which therefore delays its next use too."""
    torch = _torch()
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    here = torch.cuda.current_stream(device)
    with torch.cuda.stream(stream):
        t = torch.empty(shape, dtype=dtype, device=device)
    if here.cuda_stream != stream.cuda_stream:
        t.record_stream(here)
    return t


def kv_write(cache, batch, k, v, stream=None):
    """Quantise the batch's keys and values [tokens, heads, head_dim] into the cache."""
    if k.requires_grad or v.requires_grad:
        _no_backward()
    dtype, n, h, d = k.dtype, batch.n_tokens, cache.n_heads, cache.head_dim
    if v.dtype != dtype:
        _bad("k and v must be of one type")
    kt, kh = _rows(k, n, h, d, "k")
    vt, vh = _rows(v, n, h, d, "v")
    rc = lib().ckr_kv_write(cache._p, batch._p, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _tag(dtype), _stream_of(stream, k))
    if rc:
        _check(rc)


def kv_read(cache, batch, dtype=BF16, out=None, stream=None):
    """(k, v) of the batch's tokens as the cache holds them, [tokens, heads,
    head_dim] of dtype (a tag), into out (a pair of tensors) when given."""
    n, h, d = batch.n_tokens, cache.n_heads, cache.head_dim
    if out is None:
        out = tuple(_new((n, h, d), _torch_dtype(dtype), cache.k.device, stream) for _ in range(2))
    k, v = out
    if _tag(k.dtype) != dtype or _tag(v.dtype) != dtype:
        _bad("out must be of the type asked for")
    kt, kh = _rows(k, n, h, d, "out[0]")
    vt, vh = _rows(v, n, h, d, "out[1]")
    rc = lib().ckr_kv_read(cache._p, batch._p, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, dtype, _stream_of(stream, k))
    if rc:
        _check(rc)
    return k, v


class KvAttention:
    """Attention over a paged cache, with the workspace for batches of these sizes
    (n_heads query heads over n_kv_heads; max_context None: any).  Larger batches,
    or hints above these, are split over fewer blocks, which costs time.
    Making one waits until the workspace is zero (unless the current stream is
    being captured), so its first call may be on any stream; its calls must follow
    each other, in one stream's order or by events."""

    def __init__(self, n_heads, n_kv_heads, head_dim, n_seqs, n_tokens, max_chunk=None, max_context=None, device="cuda"):
        torch = _torch()
        self.n_heads, self.n_kv_heads, self.head_dim = int(n_heads), int(n_kv_heads), int(head_dim)
        self.ws_bytes = int(lib().ckr_kv_attention_workspace_bytes(
            self.n_heads, self.n_kv_heads, self.head_dim, n_seqs, n_tokens,
            n_tokens if max_chunk is None else max_chunk, 0xffffffff if max_context is None else max_context))
        self.ws = torch.zeros(max(self.ws_bytes, 1), dtype=torch.uint8, device=device)
        self._ws_ptr = self.ws.data_ptr()
        home = torch.cuda.current_stream(self.ws.device)
        if not torch.cuda.is_current_stream_capturing():
            home.synchronize()
        self._streams = {home.cuda_stream}   # whose work the workspace's memory outlives

    def _used_by(self, handle, stream):
        """A first call on a stream other than the one the workspace was made on."""
        torch = _torch()
        if stream is None:
            if torch.cuda.is_current_stream_capturing():   # whoever keeps the graph keeps the plan
                return
            stream = torch.cuda.current_stream(self.ws.device)
        self.ws.record_stream(stream)
        self._streams.add(handle)

    def run(self, cache, batch, q, scale=None, window=0, out=None, lse=None, stream=None):
        """Attention of the batch's tokens, whose keys and values the cache already
        holds: q [tokens, n_heads, head_dim] -> out (of q's type, new when None).
        scale: head_dim ** -0.5 when None.  lse: a contiguous float32 [tokens,
        n_heads] that receives the logarithm of each row's sum of exponentials."""
        if q.requires_grad:
            _no_backward()
        n, h, d, dtype = batch.n_tokens, self.n_heads, cache.head_dim, q.dtype
        qt, qh = _rows(q, n, h, d, "q")
        if out is None:
            out = _new(q.shape, dtype, q.device, stream)
        if out.dtype != dtype:
            _bad("out must be of q's type")
        ot, oh = _rows(out, n, h, d, "out")
        if window < 0:
            _bad("window must not be negative")
        lse_ptr = None
        if lse is not None:
            if lse.shape != q.shape[:2] or lse.dtype != _torch().float32 or not lse.is_contiguous() or not lse.is_cuda:
                _bad("lse must be a contiguous float32 [tokens, n_heads] on the GPU")
            lse_ptr = lse.data_ptr()
        handle = _stream_of(stream, q)
        if handle not in self._streams:
            self._used_by(handle, stream)
        rc = lib().ckr_kv_attention(cache._p, batch._p, q.data_ptr(), qt, qh, _tag(dtype), h, d ** -0.5 if scale is None else scale,
                                    min(window, 0xffffffff), out.data_ptr(), ot, oh, lse_ptr, self._ws_ptr, self.ws_bytes, handle)
        if rc:
            _check(rc)
        return out


def add_rms_norm(x, residual, weight, eps=1e-5, dtype=None, group=0, out=None, scales=None, total=None, stream=None):
    """h = x + residual (None: x alone), y = h / sqrt(mean(h^2) + eps) * weight over
    the last axis of x [rows, n].  Returns (out, scales, h): y of dtype (a tag; x's
    type when None, F8 or I8 with float32 scales per row, or per group of the
    row), scales None for 16 and 32 bits, h rounded to x's type.  out, scales and
    total (may be x or residual) are written in place when given.  There is no
    backward pass."""
    if x.requires_grad or weight.requires_grad or residual is not None and residual.requires_grad:
        _no_backward()
    shape, x_dtype = x.shape, x.dtype
    if len(shape) != 2:
        _bad("x must be [rows, n]")
    rows, n = shape
    xt = _tag(x_dtype)
    tag = xt if dtype is None else dtype
    coded = tag == F8 or tag == I8
    if out is None:
        out = _new(shape, _torch_dtype(tag), x.device, stream)
    if total is None:
        total = _new(shape, x_dtype, x.device, stream)
    scales_ptr = None
    if coded:
        if group < 0 or group and n % group:
            _bad("group must divide the row length")
        want = (rows, n // group) if group else (rows,)
        if scales is None:
            scales = _new(want, _torch().float32, x.device, stream)
        if scales.shape != want or scales.dtype != _torch().float32 or not scales.is_contiguous() or not scales.is_cuda:
            _bad(f"scales must be contiguous float32 {list(want)} on the GPU")
        scales_ptr = scales.data_ptr()
    elif scales is not None:
        _bad("scales belong to 8-bit outputs")
    r_ptr, rs = None, 0
    if residual is not None:
        if residual.dtype != x_dtype:
            _bad("residual must be of x's type")
        r_ptr, rs = residual.data_ptr(), _row_stride(residual, shape, "residual")
    if total.dtype != x_dtype or _tag(out.dtype) != tag:
        _bad("total must be of x's type, out of the type asked for")
    if weight.shape != shape[1:] or not weight.is_cuda or n > 1 and weight.stride(0) != 1:
        _bad(f"weight must be contiguous [{n}] on the GPU")
    rc = lib().ckr_add_rms_norm(
        x.data_ptr(), _row_stride(x, shape, "x"), r_ptr, rs, weight.data_ptr(), _tag(weight.dtype), rows, n, xt, eps, tag, group,
        out.data_ptr(), _row_stride(out, shape, "out"), scales_ptr, total.data_ptr(), _row_stride(total, shape, "total"),
        _stream_of(stream, x))
    if rc:
        _check(rc)
    return out, scales, total


def _row_stride(t, shape, what):
    if t.shape != shape or not t.is_cuda:
        _bad(f"{what} must be {list(shape)} on the GPU")
    a, b = t.stride()
    if b != 1 and shape[1] > 1:
        _bad(f"the last axis of {what} must be contiguous, {what} {list(shape)}")
    return a
