"""The operators around a 4- or 8-bit key/value cache: kv_write, kv_append, kv_read,
KvAttention, add_rms_norm and rotary over the C ABI (include/checkers_amd.h).

A KvCache names the cache's tensors, a KvBatch the tokens a call is about; both
are descriptors made once and passed to every call (the page table, starts and
offsets may change in place between calls: the kernels read them on the
device).  No call here copies or synchronises; only making a KvAttention or a
Rotary does.

stream=: the stream a call's work is queued on, None: the current one.  As with
torch's own operators the caller orders it after the streams that made the
inputs, and keeps them (or records them on it) until it is done; outputs that
a call makes belong to that stream and may be used on the current one once that
waits for it.

Only rotary has a backward pass, and a forward-mode derivative: elsewhere tensors that
require gradients are refused where gradients are recorded (not under
torch.no_grad()), and tensors with a tangent everywhere.  Calls are refused while
torch.jit.trace, make_fx or torch.export record a program, which would not hold them.
"""
import ctypes
import math

from . import CKR_E_INVALID, BF16, F16, F32, I8, CkrError, _check, _torch, lib

F8 = 16  # 8-bit floating point (e4m3, largest value 448), a type of these operators only
F4 = 17  # 4-bit floating point (e2m1, two a byte) with a power of two for each 32 values, a type of caches only

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
                      torch.float8_e4m3fn: F8, torch.float4_e2m1fn_x2: F4})
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
    and v_scale [pages, heads, page_size] in float32 (slots contiguous).  In 4 bits
    k and v are float4_e2m1fn_x2 [pages, heads, page_size, head_dim / 2] (two values an
    entry, the first in its low half), their scales float8_e8m0fnu [pages, heads,
    head_dim / 32, page_size], the last two axes contiguous."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype, "k and v must be alike, [pages, heads, page_size, head_dim]")
        _need(k.stride(3) == 1 and v.stride(3) == 1, "the last axis of k and v must be contiguous")
        self.dtype = _tag(k.dtype)
        coded = self.dtype in (F4, F8, I8)
        _need(coded == (k_scale is not None) == (v_scale is not None), "scales belong to 4- and 8-bit caches, and to both k and v")
        for t, what in ((k, "k"), (v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            if t is not None:
                _on_gpu(t, what)
                _need(t.device == k.device, "the cache's tensors must be on one GPU")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._device = k.get_device()
        self.n_pages, self.n_heads, self.page_size, row = k.shape
        self.head_dim = row * 2 if self.dtype == F4 else row
        c = _Cache(k.data_ptr(), v.data_ptr(), None, None, _i64x3(*k.stride()[:3]), _i64x3(*v.stride()[:3]),
                   _i64x2(0, 0), _i64x2(0, 0), *(int(n) for n in (k.shape[0], k.shape[2], k.shape[1], self.head_dim)),
                   self.dtype, 0)
        if self.dtype == F4:
            groups = self.head_dim // 32
            _need(groups * 32 == self.head_dim, f"head size {self.head_dim}: a multiple of 32 in 4 bits")
            for t in (k_scale, v_scale):
                _need(t.shape == (*k.shape[:2], groups, self.page_size) and t.dtype == _torch().float8_e8m0fnu and t.stride(3) == 1
                      and (groups == 1 or t.stride(2) == self.page_size),
                      "scales must be float8_e8m0fnu [pages, heads, head_dim / 32, page_size], the last two axes contiguous")
        elif coded:
            for t in (k_scale, v_scale):
                _need(t.shape == k.shape[:3] and t.dtype == _torch().float32 and t.stride(2) == 1,
                      "scales must be float32 [pages, heads, page_size], slots contiguous")
        if coded:
            c.d_k_scale, c.d_v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            c.k_scale_stride, c.v_scale_stride = _i64x2(*k_scale.stride()[:2]), _i64x2(*v_scale.stride()[:2])
        self._c = c
        self._p = ctypes.byref(c)

    @classmethod
    def empty(cls, n_pages, page_size, n_heads, head_dim, dtype, device="cuda"):
        """A cache of new tensors (dtype: F4, F8, I8, BF16 or F16), zeroed."""
        torch = _torch()
        t = _torch_dtype(dtype)
        if dtype == F4:
            _need(head_dim % 32 == 0, f"head size {head_dim}: a multiple of 32 in 4 bits")
        kv = [torch.zeros((n_pages, n_heads, page_size, head_dim // 2 if dtype == F4 else head_dim),
                          dtype=torch.uint8 if dtype in (F4, F8) else t, device=device) for _ in range(2)]
        if dtype in (F4, F8):
            kv = [x.view(t) for x in kv]
        if dtype == F4:
            sc = [torch.zeros((n_pages, n_heads, head_dim // 32, page_size), dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
                  for _ in range(2)]
        else:
            sc = [torch.zeros((n_pages, n_heads, page_size), dtype=torch.float32, device=device) if dtype in (F8, I8) else None
                  for _ in range(2)]
        return cls(kv[0], kv[1], sc[0], sc[1])

    def tensors(self):
        """The cache's tensors (k, v and, in 4 and 8 bits, their scales)."""
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
        self._device = page_table.get_device()
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


_accounts = _forward_ad = None   # torch's own of what is recorded, of the current stream, and of forward mode


def _load_accounts():
    global _accounts, _forward_ad
    torch = _torch()
    _forward_ad, c = torch.autograd.forward_ad, torch._C
    _accounts = c._get_tracing_state, c._len_torch_dispatch_stack, c._len_torch_function_stack, c._cuda_getCurrentRawStream
    return _accounts


def _not_traced():
    """Tracing (torch.jit.trace, make_fx, export) sees the output's allocation but not the call,
    so what it records would return memory that nobody writes: refused.  Other modes look on
    (and a default device, which is one as well, is told apart without asking further)."""
    traced, modes, functions, _ = _accounts
    at = _torch()._C._get_function_stack_at
    if traced() is None and not modes() and all(type(at(i)).__module__ == "torch.utils._device" for i in range(functions())):
        return
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    if traced() is not None or get_proxy_mode() is not None:
        _bad("the cache and norm operators cannot be recorded by tracing: call them outside of what is traced")


def _stream_of(stream, tensor):
    """The stream's handle; None: the current stream of the tensor's GPU.  (A
    decoding step's calls last a few microseconds each, so neither this nor the
    checks below build objects that they do not need.)"""
    traced, modes, functions, current = _accounts or _load_accounts()
    if traced() is not None or modes() or functions():
        _not_traced()
    if stream is not None:
        return stream.cuda_stream
    return current(tensor.get_device())


def _bad(msg):
    raise CkrError(CKR_E_INVALID, "[ckr] " + msg)


def _no_backward():
    """For inputs that require gradients: refused where one would be lost."""
    if _torch().is_grad_enabled():
        _bad("these operators have no backward pass: call them under torch.no_grad(), or on detached tensors")


def _tangents(*xs):
    """Whether one of the tensors carries a forward-mode tangent (torch.no_grad() keeps them)."""
    if _forward_ad is None:
        _load_accounts()
    return _forward_ad._current_level >= 0 and any(x is not None and _forward_ad.unpack_dual(x).tangent is not None for x in xs)


def _no_tangents(*xs):
    if _tangents(*xs):
        _bad("these operators have no forward-mode derivative: call them on detached tensors")


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


def _used_by(owner, tensor, handle, stream):
    """A first call on a stream other than the one an owner's tensor was made on."""
    torch = _torch()
    if stream is None:
        if torch.cuda.is_current_stream_capturing():   # whoever keeps the graph keeps its owner
            return
        stream = torch.cuda.current_stream(tensor.device)
    tensor.record_stream(stream)
    owner._streams.add(handle)


def kv_write(cache, batch, k, v, stream=None):
    """Quantise the batch's keys and values [tokens, heads, head_dim] into the cache."""
    if k.requires_grad or v.requires_grad:
        _no_backward()
    if _forward_ad is None or _forward_ad._current_level >= 0:
        _no_tangents(k, v)
    dtype, n, h, d = k.dtype, batch.n_tokens, cache.n_heads, cache.head_dim
    if v.dtype != dtype:
        _bad("k and v must be of one type")
    kt, kh = _rows(k, n, h, d, "k")
    vt, vh = _rows(v, n, h, d, "v")
    rc = lib().ckr_kv_write(cache._p, batch._p, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, _tag(dtype), _stream_of(stream, k))
    if rc:
        _check(rc)


def kv_append(cache, batch, rotary, k, v, q=None, out=None, positions=None, stream=None):
    """kv_write of keys that are turned by their positions on the way (rotary: a Rotary, which
    a captured graph needs kept; None: not turned).  q [tokens, heads, head_dim], of the keys' type: the chunk's queries,
    turned as well, into out (may be q; new when None), which is returned (None without q).
    positions: a contiguous int32 [tokens] where they are not those in the cache."""
    if k.requires_grad or v.requires_grad or q is not None and q.requires_grad:
        _no_backward()
    if _forward_ad is None or _forward_ad._current_level >= 0:
        _no_tangents(k, v, q)
    dtype, n, h, d = k.dtype, batch.n_tokens, cache.n_heads, cache.head_dim
    if v.dtype != dtype:
        _bad("k and v must be of one type")
    kt, kh = _rows(k, n, h, d, "k")
    vt, vh = _rows(v, n, h, d, "v")
    heads, q_ptr, out_ptr, qt, qh, ot, oh = 0, None, None, 0, 0, 0, 0
    if q is not None:
        if q.dtype != dtype:
            _bad("q must be of k's type")
        heads = q.shape[1] if q.dim() == 3 else 0
        qt, qh = _rows(q, n, heads, d, "q")
        if out is None:
            out = _new(q.shape, dtype, q.device, stream)
        if out.dtype != dtype:
            _bad("out must be of q's type")
        ot, oh = _rows(out, n, heads, d, "out")
        q_ptr, out_ptr = q.data_ptr(), out.data_ptr()
    elif out is not None:
        _bad("out belongs to q")
    if positions is not None and (positions.dtype != _torch().int32 or positions.shape != (n,) or not positions.is_contiguous() or not positions.is_cuda):
        _bad(f"positions must be a contiguous int32 [{n}] on the GPU")
    here = k.get_device()
    if cache._device != here or v.get_device() != here or rotary is not None and rotary._device != here or \
            batch._device != here or positions is not None and positions.get_device() != here or \
            q is not None and (q.get_device() != here or out.get_device() != here):
        _bad("the cache, the batch, the rotary and all tensors must be on one GPU")
    handle = _stream_of(stream, k)
    if rotary is not None and handle not in rotary._streams:
        _used_by(rotary, rotary.turns, handle, stream)
    rc = lib().ckr_kv_append(cache._p, batch._p, None if rotary is None else rotary._p, None if positions is None else positions.data_ptr(),
                             k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, q_ptr, qt, qh, heads, out_ptr, ot, oh, _tag(dtype),
                             handle)
    if rc:
        _check(rc)
    return out


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

    def run(self, cache, batch, q, scale=None, window=0, out=None, lse=None, stream=None):
        """Attention of the batch's tokens, whose keys and values the cache already
        holds: q [tokens, n_heads, head_dim] -> out (of q's type, new when None).
        scale: head_dim ** -0.5 when None.  lse: a contiguous float32 [tokens,
        n_heads] that receives the logarithm of each row's sum of exponentials."""
        if q.requires_grad:
            _no_backward()
        if _forward_ad is None or _forward_ad._current_level >= 0:
            _no_tangents(q)
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
            _used_by(self, self.ws, handle, stream)
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
    if _forward_ad is None or _forward_ad._current_level >= 0:
        _no_tangents(x, weight, residual)
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


# ---- rotary positions
class _Rot(ctypes.Structure):
    _fields_ = [("d_turns", ctypes.c_void_p), ("magnitude", ctypes.c_double), ("n_pairs", ctypes.c_uint32),
                ("interleaved", ctypes.c_uint32)]


def _frequencies(rotary_dim, base, scaling):
    """(radians a position of each pair, the factor on both of its values)."""
    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None:
        return f, 1.0
    s = dict(scaling)
    kind, factor = s.pop("kind", None), float(s.pop("factor", 0.0))
    known = {"linear": (), "base": (), "bands": ("length", "low", "high"), "yarn": ("length", "fast", "slow", "magnitude")}
    _need(kind in known, f"scaling kind {kind!r}: one of {', '.join(known)}")
    _need(factor > 0 and math.isfinite(factor), f"scaling factor {factor}: above 0")
    _need(set(s) <= set(known[kind]), f"scaling {kind!r} takes {', '.join(('factor',) + known[kind])}, not {', '.join(map(str, s))}")
    if kind == "linear":
        return [x / factor for x in f], 1.0
    if kind == "base":
        _need(rotary_dim > 2, "scaling 'base' needs two pairs at least")
        return [(base * factor ** (rotary_dim / (rotary_dim - 2))) ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)], 1.0
    length = float(s.get("length", 0.0))
    _need(length > 0, f"scaling {kind!r} needs the original length")
    if kind == "bands":
        low, high = float(s.get("low", 1.0)), float(s.get("high", 4.0))
        _need(high > low, f"scaling 'bands': high {high} must be above low {low}")
        keep = [min(max((length * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        return [x * (w + (1 - w) / factor) for x, w in zip(f, keep)], 1.0
    fast, slow = float(s.get("fast", 32.0)), float(s.get("slow", 1.0))
    _need(fast > slow > 0 and base > 1, "scaling 'yarn': fast above slow above 0, base above 1")
    at = [rotary_dim * math.log(length / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow)]
    lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary_dim - 1)
    ramp = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(len(f))]
    magnitude = s.get("magnitude")
    if magnitude is None:
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return [x * (1 - w) + x / factor * w for x, w in zip(f, ramp)], float(magnitude)


class Rotary:
    """How heads are turned by their positions: the pairs of a head's first rotary_dim
    values, i and i + rotary_dim / 2 (interleaved: 2 i and 2 i + 1), by position *
    frequency, that of pair i being base ** (-2 i / rotary_dim).  scaling, for contexts
    longer than a model was trained on, a dict with a "kind" and a "factor":
      linear  all frequencies / factor
      base    base * factor ** (rotary_dim / (rotary_dim - 2))
      bands   frequencies of fewer than `low` (1) turns within `length`, the original context,
              / factor, of more than `high` (4) kept, in between interpolated by their turns
      yarn    / factor and kept likewise, by a ramp over the pairs from the one of `fast` (32) turns
              within `length` to that of `slow` (1); values times `magnitude` (0.1 ln factor + 1)
    Making one copies its table to the GPU and waits for that."""

    def __init__(self, rotary_dim, base=10000.0, interleaved=False, scaling=None, device="cuda"):
        _need(rotary_dim > 0 and rotary_dim % 2 == 0, f"rotary_dim {rotary_dim}: even, from 2 on")
        _need(base > 0 and math.isfinite(base), f"base {base}: above 0")
        self._make(*_frequencies(int(rotary_dim), float(base), scaling), interleaved, device)

    @classmethod
    def of(cls, frequencies, interleaved=False, magnitude=1.0, device="cuda"):
        """One of given frequencies (radians a position, one of each pair)."""
        self = cls.__new__(cls)
        self._make([float(x) for x in frequencies], float(magnitude), interleaved, device)
        return self

    def _make(self, frequencies, magnitude, interleaved, device):
        torch = _torch()
        n = len(frequencies)
        _need(n > 0, "a rotary has one pair at least")
        _need(math.isfinite(magnitude), "the rotary's magnitude must be finite")
        self.frequencies, self.magnitude, self.interleaved, self.rotary_dim = frequencies, magnitude, bool(interleaved), 2 * n
        host = torch.empty(n, dtype=torch.int64)
        _check(lib().ckr_rotary_turns((ctypes.c_double * n)(*frequencies), n, host.data_ptr()))
        self.turns = host.to(device)   # complete when this returns
        _on_gpu(self.turns, "a rotary")
        self._device = self.turns.get_device()
        self._streams = {torch.cuda.current_stream(self.turns.device).cuda_stream}   # whose work the table outlives
        self._c = _Rot(self.turns.data_ptr(), magnitude, n, self.interleaved)
        self._p = ctypes.byref(self._c)


_i64x18, _i64x2v = ctypes.c_int64 * 18, ctypes.c_int64 * 2


def _rotate(rotary, positions, xs, outs, inverse, stream):
    """xs (one or two tensors) turned into outs."""
    q = xs[0]
    shape, dtype = q.shape, q.dtype
    four, dim = len(shape) == 4, shape[-1]
    batch, tokens = (shape[0], shape[1]) if four else (1, shape[0])
    at = positions.shape
    if len(at) == 1 and at[0] == tokens:
        ps = (0, positions.stride(0))
    elif four and len(at) == 2 and at[0] == batch and at[1] == tokens:
        ps = positions.stride()
    else:
        ps = None
    if ps is None or positions.dtype is not _torch().int32 or positions.get_device() != rotary._device:
        _bad(f"positions must be int32 {list(shape[:-2])} or {[tokens]} on the rotary's GPU")
    handle = _stream_of(stream, q)
    if handle not in rotary._streams:
        _used_by(rotary, rotary.turns, handle, stream)
    flat = []
    for i, x in enumerate(xs):
        y = outs[i]
        places = []
        for t, what in ((x, "qk"[i]), (y, "out of " + "qk"[i])):
            n = t.shape
            if len(n) != len(shape) or n[0] != shape[0] or n[-1] != dim or t.dtype is not dtype or four and n[1] != tokens or not t.is_cuda:
                _bad(f"{what} must be {[*shape[:-2], 'heads', dim]} of {dtype} on the GPU")
            st = t.stride()
            if st[-1] != 1 and t.numel():
                _bad(f"the last axis of {what} must be contiguous")
            places.append(st[:3] if four else (0, st[0], st[1]))
        if y.shape[-2] != x.shape[-2]:
            _bad(f"out of {'qk'[i]} must have its heads")
        if x.get_device() != rotary._device or y.get_device() != rotary._device:
            _bad(f"{'qk'[i]}, its output and the rotary must be on one GPU")
        flat += (x.data_ptr(), y.data_ptr(), *places[0], *places[1], x.shape[-2])
    rc = lib().ckr_rotate(rotary._p, positions.data_ptr(), _i64x2v(*ps), _i64x18(*flat), len(xs), batch, tokens, dim, _tag(dtype), inverse, handle)
    if rc:
        _check(rc)


_Turn = None


def _turn():
    """The operator with its backward pass, made when it is first needed."""
    global _Turn
    if _Turn is None:
        torch = _torch()

        class Turn(torch.autograd.Function):
            @staticmethod
            def forward(ctx, rotary, positions, inverse, *xs):
                ctx.rotary, ctx.inverse = rotary, inverse
                ctx.save_for_backward(positions)
                ctx.save_for_forward(positions)
                ctx.set_materialize_grads(False)
                outs = tuple(torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs)   # contiguous, as without gradients
                _rotate(rotary, positions, xs, outs, inverse, None)
                return outs

            @staticmethod
            def backward(ctx, *grads):
                positions, = ctx.saved_tensors
                here = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[3 + i]]
                out = [None] * len(grads)
                if here:
                    gs = [grads[i] if grads[i].stride(-1) == 1 else grads[i].contiguous() for i in here]
                    if torch.is_grad_enabled():
                        got = Turn.apply(ctx.rotary, positions, not ctx.inverse, *gs)
                    else:
                        got = [torch.empty_like(g) for g in gs]
                        _rotate(ctx.rotary, positions, gs, got, not ctx.inverse, None)
                    for i, g in zip(here, got):
                        out[i] = g
                return (None, None, None, *out)

            @staticmethod
            def jvp(ctx, _rotary, _positions, _inverse, *tangents):
                positions, = ctx.saved_tensors
                return Turn.apply(ctx.rotary, positions, ctx.inverse, *(t if t.stride(-1) == 1 else t.contiguous() for t in tangents))

        _Turn = Turn
    return _Turn


def rotary(rotary, positions, q, k=None, out=None, inverse=False, stream=None):
    """Heads turned by their tokens' positions (a Rotary): q, and k with it, [tokens, heads, dim] or
    [batch, tokens, heads, dim] with any strides but the last axis'; positions int32 [tokens] or
    [batch, tokens].  Returns the turned q, with k a pair: contiguous tensors, or into out (a tensor,
    with k a pair; may be q and k themselves) when given.  inverse turns back, but for the magnitude: it is the transposed
    matrix.  Gradients are recorded where q or k requires them, and forward-mode tangents turned
    where q or k has one (then without out and stream);
    a captured graph needs the Rotary kept, and a backward pass that is captured must not meet
    leaves of an eager graph that is still alive (torch would run their sums on its stream)."""
    xs = (q,) if k is None else (q, k)
    if not 3 <= q.dim() <= 4 or any(x.dim() != q.dim() for x in xs):
        _bad("q and k must be [tokens, heads, dim] or [batch, tokens, heads, dim]")
    tangents = (_forward_ad is None or _forward_ad._current_level >= 0) and _tangents(*xs)
    if tangents or _torch().is_grad_enabled() and any(x.requires_grad for x in xs):
        if out is not None or stream is not None:
            _bad("where gradients are recorded, or tangents turned, rotary takes neither out nor stream")
        if tangents:   # one of them may have none
            outs = tuple(_turn().apply(rotary, positions, bool(inverse), x)[0] for x in xs)
        else:
            outs = _turn().apply(rotary, positions, bool(inverse), *xs)
    else:
        if out is None:
            outs = tuple(_new(x.shape, x.dtype, x.device, stream) for x in xs)
        else:
            outs = (out,) if k is None else tuple(out)
            if len(outs) != len(xs) or any(y.requires_grad for y in outs) and _torch().is_grad_enabled():
                _bad("out must be as many tensors as are turned, and require no gradients")
        _rotate(rotary, positions, xs, outs, bool(inverse), stream)
    return outs[0] if k is None else outs
