"""kv_write, kv_read and KvAttention against plain forms: codes and scales bit for
bit, attention within bounds derived from its arithmetic."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TAGS = {"bf16": ck.BF16, "f16": ck.F16, "f32": ck.F32, "f8": ck.F8, "i8": ck.I8}


def _batch(sq, gpu, hints=True):
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)  # noqa: E731
    return ck.KvBatch(i32(sq.table), i32(sq.starts), i32(sq.offsets), sq.tokens, max(sq.lens) if hints else None,
                      max(o + n for o, n in zip(sq.starts, sq.lens)) if hints else None)


def _cache(sq, heads, dim, fmt, gpu, order="phsd", fill=None):
    """A cache whose storage has the given axis order, filled with garbage that a
    call must not use: NaN scales and codes."""
    shape = dict(p=sq.n_pages, h=heads, s=sq.page, d=dim)
    back = [order.index(c) for c in "phsd"]
    def make(t):
        x = torch.full([shape[c] for c in order], 0x7f, dtype=torch.uint8, device=gpu).view(t) if t.itemsize == 1 else \
            torch.full([shape[c] for c in order], float("nan"), dtype=t, device=gpu)
        return x.permute(back)
    t = {"f8": torch.float8_e4m3fn, "i8": torch.int8}.get(fmt) or TYPES[fmt]
    sc = [torch.full((sq.n_pages, heads, sq.page), float("nan"), device=gpu) if fmt in ko.TOP else None for _ in range(2)]
    return ck.KvCache(make(t), make(t), *sc)


def _values(cache, name, fmt):
    x = getattr(cache, name).cpu().to(torch.float64 if fmt in TYPES else torch.float32)
    if fmt in ko.TOP:
        return (x.double() * getattr(cache, name + "_scale").cpu().double()[..., None]).numpy()
    return x.numpy()


def _fill(sq, cache, batch, heads, dim, typ, gpu, seed):
    """Every token of the sequences (old and new) written; returns nothing."""
    whole = ko.Seqs([0] * len(sq.starts), [o + n for o, n in zip(sq.starts, sq.lens)], sq.page)
    whole.table = sq.table
    g = torch.Generator(device=gpu).manual_seed(seed)
    kv = [(torch.randn(whole.tokens, heads, dim, generator=g, device=gpu) * s).to(TYPES[typ]) for s in (1.3, 0.7)]
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)  # noqa: E731
    ck.kv_write(cache, ck.KvBatch(batch.page_table, i32(whole.starts), i32(whole.offsets), whole.tokens), *kv)


@pytest.mark.parametrize("fmt", ["f8", "i8", "bf16", "f16"])
@pytest.mark.parametrize("typ,heads,dim,page,order", [
    ("bf16", 8, 128, 64, "phsd"), ("f16", 3, 80, 16, "pshd"), ("f32", 1, 16, 32, "hpsd"), ("bf16", 5, 256, 16, "phsd"),
    ("f32", 2, 208, 128, "pshd"), ("f16", 7, 64, 256, "sphd")])
def test_write_and_read(gpu, fmt, typ, heads, dim, page, order):
    print(f"[case] write/read {fmt} {typ} heads={heads} dim={dim} page={page} {order}", flush=True)
    sq = ko.Seqs([5, 0, 130, 17, 0], [1, 33, 0, 100, 257], page, seed=dim)
    sq.table[3, 0] = -1 if page > 16 else sq.table[3, 0]     # an unmapped page (its tokens are not stored)
    sq.table[4, 1 if page <= 128 else 0] = sq.n_pages + 5 if page != 256 else sq.table[4, 0]
    cache = _cache(sq, heads, dim, fmt, gpu, order)
    before = [t.clone() for t in cache.tensors()]
    b = _batch(sq, gpu)
    g = torch.Generator().manual_seed(dim)
    x = [torch.randn(sq.tokens, heads, dim, generator=g) * torch.exp(3 * torch.randn(sq.tokens, heads, 1, generator=g)) for _ in range(2)]
    x[0][7] = 0                       # an empty row, a tiny one, an infinite one, one with NaN
    x[0][8] *= 0 if typ == "f16" else 1e-36
    x[1][9, 0, 3] = float("inf")
    x[1][10, heads - 1, dim - 1] = float("nan")
    x = [t.to(TYPES[typ]) for t in x]
    ck.kv_write(cache, b, *(t.to(gpu) for t in x))
    out = tuple(torch.full((sq.tokens, heads, dim), 7.0, dtype=TYPES[typ], device=gpu) for _ in range(2))
    ck.kv_read(cache, b, TAGS[typ], out=out)
    torch.cuda.synchronize()
    touched = torch.zeros(sq.n_pages, sq.page, dtype=torch.bool)
    for which, name in enumerate(("k", "v")):
        got, new = getattr(cache, name).cpu(), x[which]
        if fmt in ko.TOP:
            codes, scales = ko.quantise(new.float(), fmt)
            got_s = getattr(cache, name + "_scale").cpu()
            want_back = (codes * scales[..., None]).to(TYPES[typ])
        else:
            codes, scales, want_back = new.float().to(TYPES[fmt]), None, new.float().to(TYPES[fmt]).float().to(TYPES[typ])
        t = 0
        for s in range(len(sq.lens)):
            for i in range(sq.lens[s]):
                p, slot = sq.place(s, sq.starts[s] + i)
                if p < 0:
                    assert (out[which][t] == 0).all(), (s, i)
                    t += 1
                    continue
                touched[p, slot] = True
                have = got[p, :, slot]
                assert torch.equal(torch.nan_to_num(have.float(), nan=5e4), torch.nan_to_num(codes[t].float(), nan=5e4)), (s, i)
                if scales is not None:
                    assert torch.equal(torch.nan_to_num(got_s[p, :, slot], nan=-1.0), torch.nan_to_num(scales[t], nan=-1.0))
                back = out[which][t].cpu()
                assert torch.equal(torch.nan_to_num(back.float(), nan=5e4), torch.nan_to_num(want_back[t].float(), nan=5e4)), (s, i)
                t += 1
    for old, new in zip(before, cache.tensors()):   # nothing else was written
        keep = ~touched.to(gpu)
        a, c = (z.view(torch.uint8) if z.element_size() == 1 else z.view(torch.int16 if z.element_size() == 2 else torch.int32) for z in (old, new))
        a, c = a.transpose(1, 2)[keep], c.transpose(1, 2)[keep]
        assert torch.equal(a, c)


ATTEND = [
    # q type, cache, kv heads, group, dim, page, starts, lens, window
    ("bf16", "f8", 8, 4, 128, 64, [1000], [1], 0),
    ("bf16", "f8", 2, 4, 128, 16, [0, 5, 63, 64, 700], [1, 1, 1, 1, 1], 0),
    ("f16", "i8", 1, 8, 64, 32, [31, 32, 200], [1, 2, 1], 0),
    ("bf16", "bf16", 2, 1, 128, 128, [100, 0], [1, 1], 50),
    ("f16", "f16", 3, 2, 80, 16, [250, 0, 9], [1, 1, 5], 0),
    ("bf16", "i8", 1, 16, 256, 64, [129], [1], 0),
    ("bf16", "f8", 1, 20, 96, 16, [77, 300], [1, 1], 0),
    ("bf16", "f8", 2, 4, 128, 64, [0], [300], 0),
    ("bf16", "f8", 1, 4, 128, 32, [190, 0, 64], [70, 130, 1], 0),
    ("f16", "f16", 1, 8, 128, 16, [0, 33], [150, 64], 0),
    ("bf16", "bf16", 2, 2, 64, 256, [500], [65], 0),
    ("f16", "i8", 2, 3, 112, 64, [40, 0], [129, 31], 33),
    ("bf16", "i8", 1, 2, 256, 16, [90], [100], 0),
    ("f16", "f8", 1, 1, 16, 16, [10, 0], [40, 200], 64),
    ("bf16", "f8", 1, 7, 48, 16, [3, 0, 0, 400], [17, 0, 1, 9], 10),
    ("f16", "f16", 1, 4, 256, 32, [70, 0], [40, 90], 0),
    ("bf16", "bf16", 1, 5, 176, 16, [2000], [3], 0),
]


def _attend(gpu, typ, fmt, heads, group, dim, page, starts, lens, window, sq=None, scale=None, order="phsd", loud=1.0):
    sq = sq or ko.Seqs(starts, lens, page, seed=len(starts))
    cache = _cache(sq, heads, dim, fmt, gpu, order)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, heads, dim, typ, gpu, 3)
    g = torch.Generator(device=gpu).manual_seed(4)
    q = (torch.randn(sq.tokens, heads * group, dim, generator=g, device=gpu) * loud).to(TYPES[typ])
    plan = ck.KvAttention(heads * group, heads, dim, len(starts), sq.tokens, max(lens), max(o + n for o, n in zip(starts, lens)))
    out = torch.full_like(q, 9.0)
    lse = torch.full((sq.tokens, heads * group), 9.0, device=gpu)
    plan.run(cache, b, q, scale=scale, window=window, out=out, lse=lse)
    torch.cuda.synchronize()
    return sq, cache, b, q, plan, out, lse


def _check(sq, cache, q, out, lse, fmt, group, window, scale=None):
    D = q.shape[2]
    k, v = (np.nan_to_num(_values(cache, n, fmt), nan=0.0) for n in ("k", "v"))
    ref = ko.attention(sq, k, v, q.cpu().double().numpy(), group, scale or D ** -0.5, window)
    p_unit = ko.UNIT[q.dtype]   # weights are rounded to the queries' type
    bound, lbound = ko.attention_bounds(*ref, D, p_unit, q.dtype, np.abs(v).max())
    err = np.abs(out.cpu().double().numpy() - ref[0])
    print(f"  largest error / bound: {(err / bound).max():.3f}", flush=True)
    assert (err <= bound).all()
    got, none = lse.cpu().double().numpy(), ~np.isfinite(ref[1])
    assert (got[none] == -np.inf).all()
    assert (np.abs(got[~none] - ref[1][~none]) <= np.broadcast_to(lbound, got.shape)[~none]).all()


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c[:6])))
def test_attention(gpu, case):
    print(f"[case] attend {case}", flush=True)
    typ, fmt, heads, group, dim, page, starts, lens, window = case
    sq, cache, b, q, plan, out, lse = _attend(gpu, *case)
    _check(sq, cache, q, out, lse, fmt, group, window)
    # the same call again on the same workspace, and without hints or lse
    again = torch.full_like(q, 5.0)
    plan.run(cache, b, q, window=window, out=again)
    torch.cuda.synchronize()
    assert torch.equal(again, out)
    plan2 = ck.KvAttention(heads * group, heads, dim, len(starts), sq.tokens)
    loose = plan2.run(cache, _batch(sq, gpu, hints=False), q, window=window)
    _check(sq, cache, q, loose, lse, fmt, group, window)


@pytest.mark.parametrize("fmt", ["f8", "f16"])
@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 90, 2]])
def test_attention_unmapped_pages_and_rows_without_keys(gpu, fmt, lens):
    """Evicted pages (negative or out of range ids) are not attended to; rows whose
    window holds only such pages, or whose table is too short, give zeros and
    -inf; what lies in masked places (NaN everywhere here) never shows."""
    print(f"[case] unmapped {fmt} {lens}", flush=True)
    starts = [100, 20, 300]
    sq = ko.Seqs(starts, lens, 16, seed=8)
    full = sq.table.copy()
    cache = _cache(sq, 2, 64, fmt, gpu)
    _fill(sq, cache, _batch(sq, gpu), 2, 64, "f16", gpu, 3)
    sq.table[0, :4] = [-1, -7, sq.n_pages, 2**31 - 1]
    sq.table[1, :] = -1                      # nothing left of sequence 1
    sq.table[2, 3:17] = -1
    for s, c in ((0, 0), (0, 1), (2, 5)):    # poison the pages that went away
        cache.k[int(full[s, c])] = float("nan")
        cache.v[int(full[s, c])] = float("nan")
    g = torch.Generator(device=gpu).manual_seed(4)
    q = torch.randn(sq.tokens, 8, 64, generator=g, device=gpu).half()
    plan = ck.KvAttention(8, 2, 64, 3, sq.tokens, max(lens), 400)
    for window in (0, 30):
        lse = torch.full((sq.tokens, 8), 9.0, device=gpu)
        out = plan.run(cache, _batch(sq, gpu), q, window=window, lse=lse)
        torch.cuda.synchronize()
        assert (out[lens[0]:lens[0] + lens[1]] == 0).all()
        _check(sq, cache, q, out, lse, fmt, 4, window)
    sq.table = sq.table[:, :2].copy()        # a table narrower than the contexts
    lse = torch.full((sq.tokens, 8), 9.0, device=gpu)
    out = plan.run(cache, _batch(sq, gpu), q, lse=lse)
    torch.cuda.synchronize()
    _check(sq, cache, q, out, lse, fmt, 4, 0)


@pytest.mark.parametrize("lens", [[1], [50]])
def test_attention_poisoned_rows_show(gpu, lens):
    """A cached row that held an infinity reads as NaN: every token that sees it
    gives NaN, a token whose window ends after it does not."""
    sq = ko.Seqs([200], lens, 16, seed=1)
    cache = _cache(sq, 1, 64, "f8", gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 1, 64, "bf16", gpu, 3)
    p, slot = sq.place(0, 100)
    cache.k_scale[p, 0, slot] = float("nan")
    q = torch.randn(sq.tokens, 4, 64, device=gpu).to(torch.bfloat16)
    plan = ck.KvAttention(4, 1, 64, 1, sq.tokens, max(lens), 300)
    assert torch.isnan(plan.run(cache, b, q)).all()
    assert torch.isfinite(plan.run(cache, b, q, window=100)).all()
    cache.k_scale[p, 0, slot] = 1.0
    cache.v_scale[p, 0, slot] = float("nan")
    assert torch.isnan(plan.run(cache, b, q)).all()
    assert torch.isfinite(plan.run(cache, b, q, window=100)).all()


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("dim,group,lens,window", [(128, 4, [3, 1], 0), (64, 1, [9, 2], 5), (128, 4, [40, 20], 0), (128, 4, [100, 90], 33),
                                                   (64, 8, [70, 64], 40), (256, 2, [90, 10], 20)])
def test_infinities_and_nan_in_16_bit_values_reach_who_sees_them_only(gpu, typ, dim, group, lens, window):
    """Cached values that are infinite or NaN, in the chunk and before it: tokens
    that see them give what 32-bit sums give (infinities and NaN in those
    dimensions), tokens that do not (earlier ones, or past their window) the
    same as with finite values in their place."""
    print(f"[case] non-finite values {typ} dim={dim} group={group} {lens} window={window}", flush=True)
    sq, cache, b, q, plan, out, lse = _attend(gpu, typ, typ, 2, group, dim, 16, [50, 0], lens, window)
    clean = out.clone()
    at = [(0, 45, 0, 3, float("inf")), (0, 51, 1, dim - 1, float("nan")), (0, 50 + lens[0] // 2, 0, 0, float("-inf")),
          (0, 50 + lens[0] // 2, 0, 3, float("-inf")), (1, lens[1] - 1, 1, 7, float("inf"))]
    for s, j, h, d, x in at:
        p, slot = sq.place(s, j)
        cache.v[p, h, slot, d] = x
    got = plan.run(cache, b, q, window=window).float().cpu()
    want = clean.float().cpu()
    for s in range(2):
        for i in range(lens[s]):
            t, pos = int(sq.offsets[s]) + i, sq.starts[s] + i
            for s2, j, h, d, x in at:
                if s2 == s and j <= pos and not (window and j <= pos - window):
                    want[t, h * group:(h + 1) * group, d] += x
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    fin = torch.isfinite(want)
    # where nothing is hidden from anyone the sums are the same; values are never off by more than roundings
    assert ((got - want)[fin].abs() <= 2 * ko.UNIT[q.dtype] * want[fin].abs() + 1e-2).all()


@pytest.mark.parametrize("lens", [[1, 1], [60, 33]])
@pytest.mark.parametrize("loud,scale", [(30.0, None), (0.0, None), (1.0, -0.2), (1.0, 4.0)])
def test_attention_of_peaked_and_flat_scores(gpu, lens, loud, scale):
    print(f"[case] peaks {lens} {loud} {scale}", flush=True)
    for fmt in ("f8", "f16"):
        sq, cache, b, q, plan, out, lse = _attend(gpu, "f16", fmt, 2, 4, 128, 32, [500, 0], lens, 0, scale=scale, loud=loud)
        _check(sq, cache, q, out, lse, fmt, 4, 0, scale)


@pytest.mark.parametrize("n", [1, 70])
def test_attention_strides_and_orders(gpu, n):
    """q and out as slices of a packed projection, the cache's storage in another order."""
    sq = ko.Seqs([90, 0], [n, n], 32, seed=2)
    cache = _cache(sq, 2, 64, "i8", gpu, order="pshd")
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 64, "bf16", gpu, 3)
    big = torch.randn(sq.tokens, 3 * 8 + 5, 64, device=gpu).to(torch.bfloat16)
    q = big[:, 4:12]
    hold = torch.zeros(8, sq.tokens, 64, dtype=torch.bfloat16, device=gpu)
    lse = torch.empty(sq.tokens, 8, device=gpu)
    plan = ck.KvAttention(8, 2, 64, 2, sq.tokens)
    plan.run(cache, b, q, out=hold.transpose(0, 1), lse=lse)
    torch.cuda.synchronize()
    _check(sq, cache, q, hold.transpose(0, 1), lse, "i8", 4, 0)


def test_offsets_past_32_bits(gpu):
    """Pages whose elements lie beyond 2^32 bytes of the cache's start."""
    n_pages, page, heads, dim = 70_000, 16, 8, 512 // 4
    k = torch.zeros(n_pages, heads, page, 4 * dim, dtype=torch.int8, device=gpu)   # 4.6 GB
    cache = ck.KvCache(k[..., :dim], k[..., dim:2 * dim], *(torch.zeros(n_pages, heads, page, device=gpu) for _ in range(2)))
    sq = ko.Seqs([0], [50], page)
    sq.n_pages = n_pages
    sq.table = np.array([[n_pages - 1, n_pages - 2, 66_000, 69_000]], np.int32)
    b = _batch(sq, gpu)
    x = [torch.randn(50, heads, dim, device=gpu).half() for _ in range(2)]
    ck.kv_write(cache, b, *x)
    back = ck.kv_read(cache, b, ck.F16)
    for a, c in zip(x, back):
        codes, scales = ko.quantise(a.cpu().float(), "i8")
        assert torch.equal((codes * scales[..., None]).half(), c.cpu())
    q = torch.randn(50, heads, dim, device=gpu).half()
    lse = torch.empty(50, heads, device=gpu)
    out = ck.KvAttention(heads, heads, dim, 1, 50).run(cache, b, q, lse=lse)
    near = ko.Seqs([0], [50], page)
    near.table, near.n_pages = np.array([[3, 2, 0, 1]], np.int32), 4
    pick = torch.tensor([66_000, 69_000, n_pages - 2, n_pages - 1], device=gpu)
    small = ck.KvCache(cache.k[pick].contiguous(), cache.v[pick].contiguous(), cache.k_scale[pick].contiguous(), cache.v_scale[pick].contiguous())
    _check(near, small, q, out, lse, "i8", 1, 0)


def test_calls_on_another_stream_and_in_a_graph(gpu):
    """Write, read and attention on a side stream, then captured: every replay
    (with eager work and synchronisation between) equals the eager result, and
    follows a page table, starts and offsets changed in place."""
    sq = ko.Seqs([300, 40], [1, 1], 16, seed=5)
    cache = _cache(sq, 2, 128, "f8", gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 128, "bf16", gpu, 3)
    plan = ck.KvAttention(8, 2, 128, 2, 2, 1, 400)
    kv = [torch.randn(2, 2, 128, device=gpu).to(torch.bfloat16) for _ in range(2)]
    q, out = torch.randn(2, 8, 128, device=gpu).to(torch.bfloat16), torch.zeros(2, 8, 128, dtype=torch.bfloat16, device=gpu)
    back = tuple(torch.zeros(2, 2, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2))

    def step(stream=None):
        ck.kv_write(cache, b, *kv, stream=stream)
        ck.kv_read(cache, b, ck.BF16, out=back, stream=stream)
        plan.run(cache, b, q, out=out, stream=stream)

    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (*back, out)]
    side = torch.cuda.Stream()
    for t in (*back, out):
        t.zero_()
    torch.cuda.synchronize()
    step(side)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip((*back, out), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        for t in (*back, out):
            t.zero_()
        kv[0].copy_(torch.randn(2, 2, 128, device=gpu))
        b.starts.copy_(torch.tensor([300 - 7 * i, 40 + i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*back, out)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip((*back, out), got)), i


def test_empty_batches(gpu):
    sq = ko.Seqs([10], [2], 16)
    cache = _cache(sq, 1, 64, "f8", gpu)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    for table, starts, offsets in ((torch.zeros(0, 1, dtype=torch.int32, device=gpu), i32([]), i32([0])),
                                   (i32([[0], [1]]), i32([3, 4]), i32([0, 0, 0]))):
        b = ck.KvBatch(table, starts, offsets, 0)
        e = torch.empty(0, 1, 64, dtype=torch.bfloat16, device=gpu)
        ck.kv_write(cache, b, e, e)
        assert ck.kv_read(cache, b)[0].shape == (0, 1, 64)
        assert ck.KvAttention(4, 1, 64, 2, 0).run(cache, b, torch.empty(0, 4, 64, dtype=torch.bfloat16, device=gpu)).shape == (0, 4, 64)


def test_refusals(gpu):
    sq = ko.Seqs([10], [2], 16)
    cache = _cache(sq, 2, 64, "f8", gpu)
    b = _batch(sq, gpu)
    plan = ck.KvAttention(4, 2, 64, 1, 2)
    kv = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device=gpu)

    def bad(part, f, *a, **kw):
        with pytest.raises(ck.CkrError) as e:
            f(*a, **kw)
        assert e.value.code in (ck.CKR_E_INVALID, ck.CKR_E_CAPACITY) and part in str(e.value), str(e.value)

    bad("[2, 2, 64]", ck.kv_write, cache, b, kv[:1], kv)
    bad("one type", ck.kv_write, cache, b, kv, kv.half())
    bad("type", ck.kv_write, cache, b, kv.int(), kv.int())
    bad("contiguous", ck.kv_write, cache, b, kv.transpose(1, 2).contiguous().transpose(1, 2), kv)
    odd = torch.zeros(2 * 2 * 64 + 1, dtype=torch.bfloat16, device=gpu)[1:].view(2, 2, 64)
    bad("16-byte", ck.kv_write, cache, b, odd, kv)
    bad("16-byte", plan.run, cache, b, torch.zeros(2 * 4 * 64 + 4, dtype=torch.bfloat16, device=gpu)[4:].view(2, 4, 64))
    bad("float32, bfloat16", ck.kv_read, cache, b, ck.I8)
    bad("type", ck.kv_read, cache, b, ck.F16, out=(kv, kv))
    bad("bfloat16 or float16", plan.run, cache, b, q.float())
    bad("GPU", ck.kv_write, cache, b, kv.cpu(), kv.cpu())
    bad("lse", plan.run, cache, b, q, lse=torch.zeros(2, 4, dtype=torch.float16, device=gpu))
    bad("scale", plan.run, cache, b, q, scale=float("nan"))
    bad("window", plan.run, cache, b, q, window=-1)
    bad("multiple", ck.KvAttention(3, 2, 64, 1, 2).run, cache, b, torch.zeros(2, 3, 64, dtype=torch.bfloat16, device=gpu))
    wide = _cache(sq, 2, 64, "f16", gpu)
    bad("queries' type", plan.run, wide, b, q)
    bad("scales", ck.KvCache, cache.k, cache.v)
    bad("scales", ck.KvCache, wide.k, wide.v, cache.k_scale, cache.v_scale)
    bad("scales", ck.KvCache, cache.k, cache.v, cache.k_scale, None)
    bad("alike", ck.KvCache, cache.k, cache.v[:1], cache.k_scale, cache.v_scale)
    for shape, part in (((3, 2, 8, 64), "page size"), ((3, 2, 24, 64), "page size"), ((3, 2, 16, 40), "head size"), ((3, 2, 16, 272), "head size")):
        c = ck.KvCache(*(torch.zeros(shape, dtype=torch.float16, device=gpu) for _ in range(2)))
        bad(part, ck.kv_write, c, b, *(torch.zeros(2, 2, shape[3], dtype=torch.float16, device=gpu) for _ in range(2)))
    bad("int32", ck.KvBatch, b.page_table.long(), b.starts, b.offsets, 2)
    bad("entries", ck.KvBatch, b.page_table, b.starts, b.offsets[:1], 2)
    small = ck.KvBatch(b.page_table, b.starts, b.offsets, 2)
    small._c.d_page_table = 0x1000                     # not device memory
    bad("page table", ck.kv_write, cache, small, kv, kv)
    torch.cuda.synchronize()


@pytest.mark.parametrize("fmt", ["f8", "f16"])
def test_many_sequences_and_wrong_hints(gpu, fmt):
    """More sequences than a block has threads (some empty), one token each and
    ragged; max_chunk and max_context far from the truth on both sides."""
    r = np.random.default_rng(3)
    n = 700
    for lens in ([1] * n, [int(x) for x in r.integers(0, 4, n)]):
        starts = [int(x) for x in r.integers(0, 90, n)]
        sq = ko.Seqs(starts, lens, 16, seed=1)
        cache = _cache(sq, 1, 64, fmt, gpu)
        b = _batch(sq, gpu)
        _fill(sq, cache, b, 1, 64, "f16", gpu, 3)
        q = torch.randn(sq.tokens, 4, 64, device=gpu).half()
        plan = ck.KvAttention(4, 1, 64, n, sq.tokens)
        outs = []
        for chunk, context in ((max(lens), 100), (1, 1), (1000, 1 << 20), (40, 3)):
            print(f"[case] many sequences {fmt} hints {chunk} {context}", flush=True)
            b2 = ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, chunk, context)
            lse = torch.empty(sq.tokens, 4, device=gpu)
            outs.append(plan.run(cache, b2, q, lse=lse))
            torch.cuda.synchronize()
            if len(outs) in (1, 4):
                _check(sq, cache, q, outs[-1], lse, fmt, 4, 0)
            else:
                assert ((outs[-1].float() - outs[0].float()).abs() < 0.02).all()


def test_long_chunks_with_hints_of_one_token(gpu):
    """The kernel for few rows given long chunks, and the other way round."""
    sq = ko.Seqs([40, 0, 300], [90, 33, 1], 32, seed=1)
    for fmt, dim in (("f8", 128), ("bf16", 64), ("i8", 256)):
        cache = _cache(sq, 2, dim, fmt, gpu)
        b = _batch(sq, gpu)
        _fill(sq, cache, b, 2, dim, "bf16", gpu, 3)
        q = torch.randn(sq.tokens, 10, dim, device=gpu).to(torch.bfloat16)
        plan = ck.KvAttention(10, 2, dim, 3, sq.tokens)
        for window in (0, 50):
            for chunk in (1, 10, 500):
                print(f"[case] hints {fmt} {dim} window={window} chunk={chunk}", flush=True)
                lse = torch.empty(sq.tokens, 10, device=gpu)
                out = plan.run(cache, ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, chunk, 7), q, window=window, lse=lse)
                torch.cuda.synchronize()
                _check(sq, cache, q, out, lse, fmt, 5, window)


def test_offsets_that_are_no_batch_stay_in_bounds(gpu):
    """Chunks that overlap, run backwards or past the end: nothing outside the
    tensors is read or written, and the next call is right."""
    sq = ko.Seqs([40, 10, 60], [5, 7, 3], 16, seed=1)
    cache = _cache(sq, 1, 64, "f8", gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 1, 64, "bf16", gpu, 3)
    q = torch.randn(sq.tokens, 4, 64, device=gpu).to(torch.bfloat16)
    kv = [torch.randn(sq.tokens, 1, 64, device=gpu).to(torch.bfloat16) for _ in range(2)]
    plan = ck.KvAttention(4, 1, 64, 3, sq.tokens)
    for offsets in ([0, 15, 3, 15], [-5, 2, 100, 15], [0, 15, 0, 15], [9, 9, 9, 9]):
        for chunk in (1, 10, 100):
            print(f"[case] offsets {offsets} {chunk}", flush=True)
            bad = ck.KvBatch(b.page_table, b.starts, torch.tensor(offsets, dtype=torch.int32, device=gpu), sq.tokens, chunk, 100)
            hold = torch.full((sq.tokens + 8, 4, 64), 3.0, device=gpu).to(torch.bfloat16)
            plan.run(cache, bad, q, out=hold[4:-4])
            torch.cuda.synchronize()
            assert (hold[:4] == 3).all() and (hold[-4:] == 3).all()
            ck.kv_read(cache, bad, ck.BF16, out=(hold[4:-4, :1], hold[4:-4, 1:2]))
            torch.cuda.synchronize()
            assert (hold[:4] == 3).all() and (hold[-4:] == 3).all()
    lse = torch.empty(sq.tokens, 4, device=gpu)
    _check(sq, cache, q, plan.run(cache, b, q, lse=lse), lse, "f8", 4, 0)


def test_slots_far_apart(gpu):
    """A cache whose slots lie 80 MB from each other (offsets of a page past 32 bits),
    and one workspace for batches of several sizes."""
    far = 80 << 20
    buf = torch.empty(16 * far + (64 << 10), dtype=torch.int8, device=gpu)
    sq = ko.Seqs([20], [90], 16)
    k, v = (torch.as_strided(buf, (sq.n_pages, 2, 16, 128), (256, 128, far, 1), 32768 * i) for i in range(2))
    cache = ck.KvCache(k, v, *(torch.zeros(sq.n_pages, 2, 16, device=gpu) for _ in range(2)))
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 128, "bf16", gpu, 3)
    q = torch.randn(90, 8, 128, device=gpu).to(torch.bfloat16)
    plan = ck.KvAttention(8, 2, 128, 1, 90)
    lse = torch.empty(90, 8, device=gpu)
    _check(sq, cache, q, plan.run(cache, b, q, lse=lse), lse, "i8", 4, 0)
    for n in (1, 30, 2):
        one = ko.Seqs([20], [n], 16)
        one.table, one.n_pages = sq.table, sq.n_pages
        lse = torch.empty(n, 8, device=gpu)
        _check(one, cache, q[:n], plan.run(cache, _batch(one, gpu), q[:n], lse=lse), lse, "i8", 4, 0)


def test_one_workspace_for_calls_of_every_kind(gpu):
    """Calls that split the keys over blocks in the three ways there are, in turn on
    one workspace: each is right, and repeats bit for bit."""
    for dim in (64, 128):
        sq0 = ko.Seqs([0, 0], [700, 900], 16, seed=4)
        cache = _cache(sq0, 2, dim, "f8", gpu)
        _fill(sq0, cache, _batch(sq0, gpu), 2, dim, "bf16", gpu, 3)
        plan = ck.KvAttention(8, 2, dim, 2, 400)
        first = {}
        for turn in range(3):
            for lens in ([1, 1], [150, 90], [1, 2], [20, 30], [4, 4], [1, 1]):
                print(f"[case] one workspace dim={dim} {lens}", flush=True)
                sq = ko.Seqs([500, 800], lens, 16)
                sq.table, sq.n_pages = sq0.table, sq0.n_pages
                g = torch.Generator(device=gpu).manual_seed(sum(lens))
                q = torch.randn(sq.tokens, 8, dim, generator=g, device=gpu).to(torch.bfloat16)
                lse = torch.empty(sq.tokens, 8, device=gpu)
                out = plan.run(cache, _batch(sq, gpu), q, lse=lse)
                torch.cuda.synchronize()
                if turn == 0:
                    _check(sq, cache, q, out, lse, "f8", 4, 0)
                key = tuple(lens)
                if key in first:
                    assert torch.equal(first[key][0], out) and torch.equal(first[key][1], lse)
                first.setdefault(key, (out, lse))


def _raw(t):
    """The bytes of a tensor (NaN equal to itself)."""
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16 if t.element_size() == 2 else torch.int32)


@pytest.mark.parametrize("rows", ["one", "shifted"])
@pytest.mark.parametrize("n", [1, 30])
def test_page_tables_whose_rows_overlap(gpu, rows, n):
    """One row of pages for all sequences (stride 0), and rows that start a page
    further on each (stride 1): as the same rows apart, with page numbers of
    other sequences right behind the table."""
    starts, page, S = [0, 40, 90], 16, 3
    hold = torch.tensor([7, 3, 11, 0, 5, 9, 2, 8, 1, 13, 4, 12] + [6, 10, 14] * 20, dtype=torch.int32, device=gpu)
    width = 9
    table = hold[:width].expand(S, width) if rows == "one" else torch.as_strided(hold, (S, width), (1, 1))
    apart = table.contiguous()
    assert apart.stride(0) == width and not table.is_contiguous()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    b, c = (ck.KvBatch(t, i32(starts), i32([n * s for s in range(S + 1)]), S * n, n, 90 + n) for t in (table, apart))
    g = torch.Generator(device=gpu).manual_seed(n)
    kv = [torch.randn(S * n, 2, 64, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2)]
    q = torch.randn(S * n, 8, 64, generator=g, device=gpu).to(torch.bfloat16)
    plan, got = ck.KvAttention(8, 2, 64, S, S * n, n, 200), []
    for batch in (b, c):
        cache = ck.KvCache.empty(15, page, 2, 64, ck.F8, device=gpu)
        old = [torch.randn(15, 2, page, 64, generator=torch.Generator(device=gpu).manual_seed(s), device=gpu) for s in (5, 6)]
        every = ck.KvBatch(torch.arange(15, dtype=torch.int32, device=gpu)[None], i32([0]), i32([0, 15 * page]), 15 * page)
        ck.kv_write(cache, every, *(x.transpose(1, 2).reshape(-1, 2, 64) for x in old))
        ck.kv_write(cache, batch, *kv)
        got.append([*(t.clone() for t in cache.tensors()), *ck.kv_read(cache, batch), plan.run(cache, batch, q)])
    torch.cuda.synchronize()
    for x, y in zip(*got):
        assert torch.equal(_raw(x), _raw(y))


def _busy(ms=40):
    """Work of about so long on the current stream."""
    torch.cuda._sleep(int(ms * 1.5e6))


def _decoding(gpu):
    """A decoding step whose items are shared by blocks: (cache, batch, q, sizes of
    its plan, what it gives)."""
    sq = ko.Seqs([900, 400], [1, 1], 16, seed=5)
    cache = _cache(sq, 2, 128, "f8", gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 128, "bf16", gpu, 3)
    q = torch.randn(2, 8, 128, device=gpu).to(torch.bfloat16)
    sizes = (8, 2, 128, 2, 2, 1, 901)
    want = ck.KvAttention(*sizes).run(cache, b, q)
    torch.cuda.synchronize()
    return cache, b, q, sizes, want


@pytest.mark.parametrize("explicit", [True, False])
def test_plan_made_behind_queued_work_and_run_at_once_on_another_stream(gpu, explicit):
    """The workspace's memory held other bytes before; the first call, on a stream that
    waits for nothing, finds zeros."""
    cache, b, q, sizes, want = _decoding(gpu)
    side, out = torch.cuda.Stream(), torch.zeros_like(q)
    n = ck.KvAttention(*sizes).ws.numel()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    dirty = torch.full((n,), 0x5a, dtype=torch.uint8, device=gpu)
    torch.cuda.synchronize()
    del dirty
    _busy()
    plan = ck.KvAttention(*sizes)
    if explicit:
        plan.run(cache, b, q, out=out, stream=side)
    else:
        with torch.cuda.stream(side):
            plan.run(cache, b, q, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    assert (plan.ws[:2048] == 0).all()   # the counters, as the next call needs them


@pytest.mark.parametrize("explicit", [True, False])
def test_plan_dropped_while_another_stream_runs_it(gpu, explicit):
    """Its workspace is not handed out before that call has ended."""
    cache, b, q, sizes, want = _decoding(gpu)
    side, out = torch.cuda.Stream(), torch.zeros_like(q)
    plan = ck.KvAttention(*sizes)
    n, at = plan.ws.numel(), plan.ws.data_ptr()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        _busy()
        if not explicit:
            plan.run(cache, b, q, out=out)
    if explicit:
        plan.run(cache, b, q, out=out, stream=side)
    del plan
    other = torch.full((n,), 0x5a, dtype=torch.uint8, device=gpu)
    assert other.data_ptr() != at
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and (other == 0x5a).all()


def _calls_that_make_outputs(gpu):
    """Calls by name, each giving the tensors that it made, on a given stream."""
    sq = ko.Seqs([90], [1000], 16, seed=5)
    cache = _cache(sq, 2, 64, "f8", gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 64, "bf16", gpu, 3)
    q = torch.randn(sq.tokens, 8, 64, device=gpu).to(torch.bfloat16)
    x, w = torch.randn(1000, 1024, device=gpu).to(torch.bfloat16), torch.ones(1024, device=gpu).to(torch.bfloat16)
    plan = ck.KvAttention(8, 2, 64, 1, sq.tokens, sq.tokens, 1090)
    return {"read": lambda s: list(ck.kv_read(cache, b, stream=s)), "attend": lambda s: [plan.run(cache, b, q, stream=s)],
            "norm": lambda s: list(ck.add_rms_norm(x, None, w, dtype=ck.F8, stream=s))}


@pytest.mark.parametrize("name", ["read", "attend", "norm"])
def test_outputs_made_for_another_stream_are_not_memory_still_read_here(gpu, name):
    call, side = _calls_that_make_outputs(gpu)[name], torch.cuda.Stream()
    want = call(None)
    torch.cuda.synchronize()
    held = [torch.full((t.numel() * t.element_size(),), 0x5a, dtype=torch.uint8, device=gpu) for t in want]
    copies = [torch.zeros_like(t) for t in held]
    at = {t.data_ptr() for t in held}
    torch.cuda.synchronize()
    _busy()
    for t, c in zip(held, copies):
        c.copy_(t)                     # still to come when the block is given back
    del held, t
    got = call(side)
    assert not at & {t.data_ptr() for t in got}
    side.synchronize()
    assert all(torch.equal(_raw(x), _raw(y)) for x, y in zip(got, want))
    torch.cuda.synchronize()
    assert all((c == 0x5a).all() for c in copies)


@pytest.mark.parametrize("name", ["read", "attend", "norm"])
def test_outputs_made_for_another_stream_and_dropped_here_are_kept_until_read(gpu, name):
    call, side = _calls_that_make_outputs(gpu)[name], torch.cuda.Stream()
    want = call(None)
    torch.cuda.synchronize()
    got = call(side)
    at = {t.data_ptr() for t in got}
    torch.cuda.current_stream().wait_stream(side)
    _busy()
    copies = [_raw(t).clone() for t in got]
    del got
    with torch.cuda.stream(side):
        other = [torch.full_like(_raw(t), 0x5a) for t in want]
    assert not at & {t.data_ptr() for t in other}
    torch.cuda.synchronize()
    assert all(torch.equal(x, _raw(y)) for x, y in zip(copies, want))


@pytest.mark.parametrize("fmt", ["f8", "f16"])
@pytest.mark.parametrize("lens", [[1, 1], [3, 8], [9, 20], [70, 90]])
def test_plans_smaller_than_the_batch_or_its_hints(gpu, fmt, lens):
    """A plan for short contexts given a wide table and no hints, and one for a single
    token: less of a split, the same answer."""
    sq = ko.Seqs([700, 300], lens, 16, seed=4, width=5000)
    cache = _cache(sq, 2, 128, fmt, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 128, "f16", gpu, 3)
    q = torch.randn(sq.tokens, 8, 128, device=gpu).half()
    chunk = max(lens)
    for sizes in ((8, 2, 128, 2, sq.tokens, chunk, 100), (8, 2, 128, 1, 1, 1, 1), (8, 2, 128, 2, sq.tokens, chunk, 1000)):
        plan = ck.KvAttention(*sizes)
        for context in (None, 1 << 16, 1000):
            print(f"[case] small plans {fmt} {lens} {sizes[3:]} context={context}", flush=True)
            lse = torch.empty(sq.tokens, 8, device=gpu)
            out = plan.run(cache, ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, chunk, context), q, lse=lse)
            torch.cuda.synchronize()
            _check(sq, cache, q, out, lse, fmt, 4, 0)
            assert (plan.ws[:2048] == 0).all()
    if chunk == 1:
        plan.ws_bytes = 2048
        with pytest.raises(ck.CkrError) as e:
            plan.run(cache, b, q)
        assert e.value.code == ck.CKR_E_CAPACITY


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [48, 80, 112, 128, 208])
def test_an_infinite_key_weighs_nothing_where_its_score_is_minus_infinity(gpu, typ, dim):
    """An infinity in a key's last dimension, seen with a score of -infinity: as if
    the key were not there, by each of the kernels that hints choose."""
    sq = ko.Seqs([100], [90], 16, seed=2)
    cache = _cache(sq, 1, dim, typ, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 1, dim, typ, gpu, 3)
    q = torch.randn(90, 8, dim, device=gpu).to(TYPES[typ])
    q[..., dim - 1] = -q[..., dim - 1].abs() - 0.25
    p, slot = sq.place(0, 37)
    for inf in (False, True):
        cache.k[p, 0, slot, dim - 1] = float("inf") if inf else 0
        k = _values(cache, "k", typ)
        if inf:   # a finite stand-in: its weight is 0 in 64 bits too
            k[p, 0, slot] = 0
            k[p, 0, slot, dim - 1] = 1e9
        for chunk in (1, 10, 90):
            print(f"[case] infinite key {typ} {dim} {inf} chunk={chunk}", flush=True)
            lse = torch.empty(90, 8, device=gpu)
            plan = ck.KvAttention(8, 1, dim, 1, 90)
            out = plan.run(cache, ck.KvBatch(b.page_table, b.starts, b.offsets, 90, chunk, 200), q, lse=lse)
            torch.cuda.synchronize()
            v = np.nan_to_num(_values(cache, "v", typ))
            ref = ko.attention(sq, np.nan_to_num(k), v, q.cpu().double().numpy(), 8, dim ** -0.5, 0)
            if not inf:
                slack = ref[3]
            ref = (*ref[:3], slack, ref[4])   # the stand-in's own products are not what the kernels round
            bound, lbound = ko.attention_bounds(*ref, dim, ko.UNIT[q.dtype], q.dtype, np.abs(v).max())
            assert (np.abs(out.cpu().double().numpy() - ref[0]) <= bound).all()
            assert (np.abs(lse.cpu().double().numpy() - ref[1]) <= lbound).all()


@pytest.mark.parametrize("typ", ["bf16", "f16"])
@pytest.mark.parametrize("fmt", ["f8", "i8"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
def test_the_log_sum_does_not_depend_on_the_values(gpu, typ, fmt, dim, page):
    """Value rows of scale NaN: NaN for who sees them, with the log-sum of the scores
    all the same; for who does not, nothing changes.  By each of the kernels."""
    sq = ko.Seqs([300, 40], [90, 7], page, seed=2)
    cache = _cache(sq, 2, dim, fmt, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, dim, typ, gpu, 3)
    q = torch.randn(97, 8, dim, device=gpu).to(TYPES[typ])
    at = ((0, 3, 0), (0, 350, 1), (1, 41, 1))
    for chunk in (1, 10, 90):
        b2 = ck.KvBatch(b.page_table, b.starts, b.offsets, 97, chunk, 400)
        plan = ck.KvAttention(8, 2, dim, 2, 97)
        for window in (0, 300):
            print(f"[case] log-sum {typ} {fmt} {dim} {page} chunk={chunk} window={window}", flush=True)
            lse0, lse = (torch.empty(97, 8, device=gpu) for _ in range(2))
            clean = plan.run(cache, b2, q, window=window, lse=lse0)
            held = cache.v_scale.clone()
            for s, j, h in at:
                p, slot = sq.place(s, j)
                cache.v_scale[p, h, slot] = float("nan")
            got = plan.run(cache, b2, q, window=window, lse=lse)
            cache.v_scale.copy_(held)
            sees = torch.zeros(97, 8, dtype=torch.bool, device=gpu)
            for s, j, h in at:
                for i in range(sq.lens[s]):
                    pos = sq.starts[s] + i
                    if j <= pos and not (window and j <= pos - window):
                        sees[int(sq.offsets[s]) + i, 4 * h:4 * h + 4] = True
            assert torch.isnan(got[sees]).all()
            assert torch.equal(got[~sees], clean[~sees])
            assert torch.equal(lse, lse0)


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (80, 32), (256, 16)])
@pytest.mark.parametrize("x", [float("inf"), float("-inf")])
def test_an_infinity_that_every_row_sees_with_a_small_weight(gpu, dim, page, x):
    """float16 values: an infinity in a tile that every row sees wholly, whose weight
    (2^-45 of the largest, 2^-60) is 0 in 16 bits and not in 32: an infinity, by
    each of the kernels that hints choose; rows that do not see it are as before."""
    sq = ko.Seqs([300], [90], page, seed=2)
    cache = _cache(sq, 1, dim, "f16", gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 1, dim, "f16", gpu, 3)
    cache.k[..., 0] = torch.where(torch.isnan(cache.k[..., 0]), cache.k[..., 0], 2.0)
    q = torch.zeros(90, 8, dim, dtype=torch.float16, device=gpu)
    q[..., 0] = 16.0
    scale = 0.2                            # a key's weight: exp(0.2 * 16 * its first element)
    for j, first in ((5, -7.75), (131, -11.0)):
        p, slot = sq.place(0, j)
        cache.k[p, 0, slot, 0] = first
    for chunk in (1, 10, 90):
        b2 = ck.KvBatch(b.page_table, b.starts, b.offsets, 90, chunk, 400)
        plan = ck.KvAttention(8, 1, dim, 1, 90)
        for window in (0, 260):
            print(f"[case] small weight {dim} {page} {x} chunk={chunk} window={window}", flush=True)
            lse0, lse = (torch.empty(90, 8, device=gpu) for _ in range(2))
            clean = plan.run(cache, b2, q, scale=scale, window=window, lse=lse0).float().cpu()
            held = cache.v.clone()
            for j, d in ((5, 3), (131, dim - 1)):
                p, slot = sq.place(0, j)
                cache.v[p, 0, slot, d] = x
            got = plan.run(cache, b2, q, scale=scale, window=window, lse=lse).float().cpu()
            cache.v.copy_(held)
            want = clean.clone()
            for t in range(90):
                for j, d in ((5, 3), (131, dim - 1)):
                    if not window or j > 300 + t - window:
                        want[t, :, d] = x
            inf = torch.isinf(want)
            assert torch.equal(got[inf], want[inf])
            # the rest: weights in 16 bits of other sums' maxima, roundings only
            assert ((got - want)[~inf].abs() <= 2 * ko.UNIT[torch.float16] * want[~inf].abs() + 2.0 ** -24).all()
            # both within their bound of the exact one: scores up to 0.2 * 16 * 11
            assert ((lse - lse0).abs() <= 2 * ko.U32 * ((dim + 8) * 36 + (400 + 16) + 4 * (1 + lse0.abs()))).all()


def test_calls_that_would_lose_a_gradient_are_refused(gpu):
    sq = ko.Seqs([10], [2], 16)
    cache = _cache(sq, 2, 64, "f8", gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 64, "bf16", gpu, 3)
    kv, q = (torch.randn(2, h, 64, device=gpu).to(torch.bfloat16) for h in (2, 4))
    plan = ck.KvAttention(4, 2, 64, 1, 2)
    kv2, q2 = (t.clone().requires_grad_() for t in (kv, q))
    for f, a in ((ck.kv_write, (cache, b, kv2, kv)), (ck.kv_write, (cache, b, kv, kv2)), (plan.run, (cache, b, q2))):
        with pytest.raises(ck.CkrError) as e:
            f(*a)
        assert e.value.code == ck.CKR_E_INVALID and "no backward" in str(e.value)
    with torch.no_grad():
        ck.kv_write(cache, b, kv2, kv2)
        got = plan.run(cache, b, q2)
    assert torch.equal(got, plan.run(cache, b, q))


def test_axes_of_one_entry_may_have_any_stride(gpu):
    """One token, one head, one page, one sequence, one column of pages: their
    strides are never taken."""
    def odd(t, *axes):
        return torch.as_strided(t, t.shape, [3 if i in axes else s for i, s in enumerate(t.stride())], t.storage_offset())

    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    kv = [torch.randn(1, 1, 64, device=gpu).half() for _ in range(2)]
    q = torch.randn(1, 1, 64, device=gpu).half()
    for fmt in (ck.I8, ck.F16):
        got = []
        for strange in (False, True):
            cache = ck.KvCache.empty(1, 16, 1, 64, fmt, device=gpu)
            b = ck.KvBatch(i32([[0]]), i32([5]), i32([0, 1]), 1)
            k, v, x = *kv, q
            if strange:
                cache = ck.KvCache(*(odd(t, 0, 1) for t in cache.tensors()))
                b = ck.KvBatch(odd(i32([[0]]), 0, 1), i32([5]), i32([0, 1]), 1)
                k, v, x = (odd(t, 0, 1) for t in (k, v, x))
            ck.kv_write(cache, b, k, v)
            out = torch.empty(1, 1, 64, device=gpu).half()
            back = ck.kv_read(cache, b, ck.F16, out=tuple(odd(torch.empty_like(out), 0, 1) if strange else torch.empty_like(out) for _ in range(2)))
            ck.KvAttention(1, 1, 64, 1, 1).run(cache, b, x, out=odd(out, 0, 1) if strange else out)
            got.append([t.clone() for t in (*cache.tensors(), *back, out)])
        torch.cuda.synchronize()
        assert all(torch.equal(_raw(s.contiguous()), _raw(t.contiguous())) for s, t in zip(*got))
    table = torch.stack([i32([3, 1, 2]), i32([0, 0, 0])], 1)[:, :1]     # one column, stride 2
    seqs = ck.KvBatch(table, i32([0, 0, 0]), i32([0, 1, 2, 3]), 3)
    cache = ck.KvCache.empty(4, 16, 1, 64, ck.F16, device=gpu)
    x = torch.randn(3, 1, 64, device=gpu).half()
    ck.kv_write(cache, seqs, x, x)
    assert torch.equal(cache.k[[3, 1, 2], 0, 0], x[:, 0])
    turned = ck.KvBatch(torch.stack([i32([3]), i32([0])], 1)[0, :].view(1, 2).t()[:1], i32([0]), i32([0, 1]), 1)
    assert torch.equal(ck.kv_read(cache, turned, ck.F16)[0], x[:1])


def test_outputs_whose_rows_overlap_are_refused(gpu):
    """What is written twice would hold either; what is only read may overlap."""
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    b = ck.KvBatch(i32([[1]]), i32([5]), i32([0, 2]), 2)
    kv, q = torch.randn(2, 2, 64, device=gpu).half(), torch.randn(2, 4, 64, device=gpu).half()
    cache = ck.KvCache.empty(3, 16, 2, 64, ck.I8, device=gpu)
    ck.kv_write(cache, b, kv[:, :1].expand(2, 2, 64), kv[:1].expand(2, 2, 64))
    plan = ck.KvAttention(4, 2, 64, 1, 2)

    def bad(f, *a, **kw):
        with pytest.raises(ck.CkrError) as e:
            f(*a, **kw)
        assert e.value.code == ck.CKR_E_INVALID and "overlap" in str(e.value), str(e.value)

    rows = torch.empty(2, 4, 64, device=gpu).half()
    for t in (rows[:1].expand(2, 4, 64), rows[:, :1].expand(2, 4, 64), torch.as_strided(rows, (2, 4, 64), (64, 64, 1)),
              torch.as_strided(rows, (2, 4, 64), (256, 32, 1))):
        bad(plan.run, cache, b, q, out=t)
        bad(ck.kv_read, cache, b, ck.F16, out=(t[:, :2], torch.empty_like(kv)))
        bad(ck.kv_read, cache, b, ck.F16, out=(torch.empty_like(kv), t[:, :2]))
    plan.run(cache, b, q, out=torch.empty(4, 2, 64, device=gpu).half().transpose(0, 1))
    # one head's keys and values for all heads: read by the attention, not written
    k, v, ks, vs = cache.tensors()
    shared = ck.KvCache(k[:, :1].expand(k.shape), v[:, :1].expand(v.shape), ks[:, :1].expand(ks.shape), vs[:, :1].expand(vs.shape))
    got = plan.run(shared, b, q)
    one = ck.KvCache(*(t[:, :1] for t in cache.tensors()))
    assert torch.equal(got, ck.KvAttention(4, 1, 64, 1, 2).run(one, b, q))
    bad(ck.kv_write, shared, b, kv, kv)
    bad(ck.kv_write, ck.KvCache(k, v, ks, vs[:1].expand(vs.shape)), b, kv, kv)
    bad(ck.kv_write, ck.KvCache(k, v[:1].expand(v.shape), ks, vs), b, kv, kv)
    torch.cuda.synchronize()


@pytest.mark.parametrize("lens", [[1, 1], [20, 9], [90, 40]])
def test_windows_longer_than_any_context(gpu, lens):
    """As no window; 2^32 + 5 is not a window of 5."""
    sq, cache, b, q, plan, out, lse = _attend(gpu, "bf16", "f8", 2, 4, 64, 16, [100, 30], lens, 0)
    for window in ((1 << 31) - 1, (1 << 32) - 1, 1 << 32, (1 << 32) + 5, 1 << 40):
        got = plan.run(cache, b, q, window=window)
        assert torch.equal(got, out), window


def test_overlapping_chunks_whose_tiles_exceed_32_bits(gpu):
    """2500 sequences that each claim the whole of 1000 rows behind a million unmapped
    keys: 4.9e9 key tiles in all.  Nothing outside the tensors is touched, and the
    next call is right."""
    n, tokens, page = 5000, 1000, 256
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    cache = ck.KvCache.empty(2, page, 1, 64, ck.F8, device=gpu)
    table = torch.full((1, 4096), -1, dtype=torch.int32, device=gpu).expand(n, 4096)
    ends = [0 if i % 2 == 0 else tokens for i in range(n + 1)]
    starts = torch.full((n,), 1_000_000, dtype=torch.int32, device=gpu)
    q = torch.randn(tokens, 1, 64, device=gpu).to(torch.bfloat16)
    plan = ck.KvAttention(1, 1, 64, n, tokens, 1, 1 << 20)
    hold = torch.full((tokens + 64, 1, 64), 3.0, device=gpu).to(torch.bfloat16)
    for offsets in (ends, [0] + [tokens] * n):
        print("[case] overlapping chunks", offsets[:3], flush=True)
        plan.run(cache, ck.KvBatch(table, starts, i32(offsets), tokens, 1, 1 << 20), q, out=hold[32:-32])
        torch.cuda.synchronize()
        assert (hold[:32] == 3).all() and (hold[-32:] == 3).all()
        assert (plan.ws[:2048] == 0).all()
    sq, cache, b, q, _, out, lse = _attend(gpu, "bf16", "f8", 1, 1, 64, 16, [100, 30], [1, 1], 0)
    assert torch.equal(plan.run(cache, b, q), ck.KvAttention(1, 1, 64, n, tokens, 1, 1 << 20).run(cache, b, q))
    _check(sq, cache, q, plan.run(cache, b, q, lse=lse), lse, "f8", 1, 0)


@pytest.mark.parametrize("kernel,starts,lens", [("wide", [1300, 1531], [70, 66]), ("many", [1300, 1531], [20, 9]), ("few", [5300, 4531], [3, 8])])
@pytest.mark.parametrize("typ,fmt", [("bf16", "f8"), ("bf16", "bf16"), ("f16", "i8"), ("f16", "f8"), ("f16", "f16")])
@pytest.mark.parametrize("page,dim", [(16, 128), (64, 128), (256, 64), (32, 64), (128, 256)])
def test_long_contexts_in_one_piece(gpu, kernel, starts, lens, typ, fmt, page, dim):
    """Twenty key tiles and more in one block (a context hint of 1 splits nothing, and
    gives few rows two blocks), so that what the kernels load ahead comes round
    several times: plain, with a window, with a page gone from the middle, and with
    scores that rise along the context, so that the maximum moves late too."""
    group = 4
    sq = ko.Seqs(starts, lens, page, seed=page)
    cache = _cache(sq, 1, dim, fmt, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 1, dim, typ, gpu, 3)
    near = ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, max(lens), 1)
    g = torch.Generator(device=gpu).manual_seed(4)
    q = torch.randn(sq.tokens, group, dim, generator=g, device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(group, 1, dim, 2, sq.tokens, max(lens), 1)

    def check(what, batch, qq, window=0):
        print(f"[case] one piece {kernel} {typ} {fmt} page={page} {what}", flush=True)
        lse = torch.empty(sq.tokens, group, device=gpu)
        out = plan.run(cache, batch, qq, window=window, lse=lse)
        torch.cuda.synchronize()
        _check(sq, cache, qq, out, lse, fmt, group, window)

    check("plain", near, q)
    check("window", near, q, 700)
    table = sq.table.copy()
    sq.table[0, 640 // page] = -1
    sq.table[1, 1100 // page] = sq.n_pages
    i32 = torch.tensor(sq.table, dtype=torch.int32, device=gpu)
    check("hole", ck.KvBatch(i32, b.starts, b.offsets, sq.tokens, max(lens), 1), q)
    sq.table = table
    # keys whose first element grows by 0.04 a position, queries with 8 there
    whole = ko.Seqs([0, 0], [o + n for o, n in zip(starts, lens)], page)
    ramp = torch.cat([torch.arange(n, device=gpu) * 0.04 for n in whole.lens])
    k, v = (torch.randn(whole.tokens, 1, dim, generator=g, device=gpu) for _ in range(2))
    k[:, 0, 0] = ramp
    every = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in (whole.starts, whole.offsets)]
    ck.kv_write(cache, ck.KvBatch(b.page_table, *every, whole.tokens), k.to(TYPES[typ]), v.to(TYPES[typ]))
    q = q.clone()
    q[..., 0] = 8
    check("rising", near, q)


@pytest.mark.parametrize("typ,fmt", [("bf16", "f8"), ("bf16", "bf16"), ("bf16", "i8"), ("f16", "i8"), ("f16", "f16")])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (96, 32), (256, 16)])
def test_weights_of_few_rows_hold_twice_the_bits(gpu, typ, fmt, dim, page):
    """Two products a value: the sums' error is that of 16 bits (bfloat16) or 22, a small
    part of what one rounding to 8 or 11 gives where the values cancel."""
    case = (typ, fmt, 2, 4, dim, page, [1500, 700, 31], [1, 1, 2], 0)
    sq, cache, b, q, plan, out, lse = _attend(gpu, *case)
    k, v = (np.nan_to_num(_values(cache, n, fmt), nan=0.0) for n in ("k", "v"))
    ref = ko.attention(sq, k, v, q.cpu().double().numpy(), 4, dim ** -0.5, 0)
    bound, _ = ko.attention_bounds(*ref, dim, ko.UNIT[q.dtype] ** 2, q.dtype, np.abs(v).max())
    err = np.abs(out.cpu().double().numpy() - ref[0])
    print(f"  largest error / bound: {(err / bound).max():.3f}", flush=True)
    assert (err <= bound).all()


@pytest.mark.parametrize("fmt", ["f8", "i8"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 32)])
@pytest.mark.parametrize("spread", [0, 4, 30])
def test_bfloat16_queries_over_8_bits_keep_11_bits_of_the_weights(gpu, fmt, dim, page, spread):
    """Through each kernel, over contexts in one piece and split; with value rows whose
    magnitudes differ by up to 2^60, some of them zero, growing along one context."""
    starts, lens, group = [900, 0], [70, 45], 4
    sq = ko.Seqs(starts, lens, page, seed=page)
    cache = _cache(sq, 1, dim, fmt, gpu)
    b = _batch(sq, gpu)
    whole = ko.Seqs([0, 0], [o + n for o, n in zip(starts, lens)], page)
    g = torch.Generator(device=gpu).manual_seed(9)
    k, v = (torch.randn(whole.tokens, 1, dim, generator=g, device=gpu) for _ in range(2))
    if spread:
        powers = (torch.rand(whole.tokens, 1, 1, generator=g, device=gpu) * 2 * spread - spread).round()
        powers[:whole.lens[0]] = powers[:whole.lens[0]].sort(0).values if spread == 4 else powers[:whole.lens[0]]
        v *= torch.exp2(powers)
        v[3::17] = 0
    every = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in (whole.starts, whole.offsets)]
    ck.kv_write(cache, ck.KvBatch(b.page_table, *every, whole.tokens), k, v)
    q = (torch.randn(sq.tokens, group, dim, generator=g, device=gpu) * 1.5).to(torch.bfloat16)
    kd, vd = (np.nan_to_num(_values(cache, n, fmt), nan=0.0) for n in ("k", "v"))
    ref = ko.attention(sq, kd, vd, q.cpu().double().numpy(), group, dim ** -0.5, 0)
    # a weight with its value's scale rounds by 2^-25 at least, held against 2^6 of the largest scale: 2^-31 of the largest value
    bound, lbound = ko.attention_bounds(*ref, dim, ko.UNIT[torch.float16], q.dtype, 2 * np.abs(vd).max())
    for chunk in (70, 20, 1):
        for context in (1, 1000):
            print(f"[case] 11 bits {fmt} {dim} spread={spread} chunk={chunk} context={context}", flush=True)
            lse = torch.empty(sq.tokens, group, device=gpu)
            plan = ck.KvAttention(group, 1, dim, 2, sq.tokens, chunk, context)
            out = plan.run(cache, ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, chunk, context), q, lse=lse)
            torch.cuda.synchronize()
            err = np.abs(out.cpu().double().numpy() - ref[0])
            print(f"  largest error / bound: {(err / bound).max():.3f}", flush=True)
            assert (err <= bound).all()
            assert (np.abs(lse.cpu().double().numpy() - ref[1]) <= lbound).all()
