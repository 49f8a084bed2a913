"""A cache in 4 bits: kv_write, kv_read and KvAttention against plain forms, codes and
powers exactly, attention within bounds derived from its arithmetic."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests import kv4_oracle as k4
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TAGS = {"bf16": ck.BF16, "f16": ck.F16, "f32": ck.F32}


def _i32(a, gpu):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)


def _batch(sq, gpu, hints=True):
    return ck.KvBatch(_i32(sq.table, gpu), _i32(sq.starts, gpu), _i32(sq.offsets, gpu), sq.tokens, max(sq.lens) if hints else None,
                      max(o + n for o, n in zip(sq.starts, sq.lens)) if hints else None)


def _cache(sq, heads, dim, gpu, order="phsd", garbage=True):
    """A cache whose storage has the given axis order, filled with what a call must not
    use: codes of 6 and powers of NaN."""
    shape = dict(p=sq.n_pages, h=heads, s=sq.page, d=dim // 2)
    back = [order.index(c) for c in "phsd"]
    kv = [torch.full([shape[c] for c in order], 0x77 if garbage else 0, dtype=torch.uint8, device=gpu).permute(back).view(torch.float4_e2m1fn_x2)
          for _ in range(2)]
    sc = [torch.full((sq.n_pages, heads, dim // 32, sq.page), 255 if garbage else 0, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu)
          for _ in range(2)]
    return ck.KvCache(*kv, *sc)


def _bytes(t):
    return t.view(torch.uint8)


def _values(cache, name):
    return k4.values(_bytes(getattr(cache, name)).cpu(), _bytes(getattr(cache, name + "_scale")).cpu())


def _fill(sq, cache, batch, heads, dim, gpu, seed, scale=(1.3, 0.7)):
    """Every token of the sequences (old and new) written."""
    whole = ko.Seqs([0] * len(sq.starts), [o + n for o, n in zip(sq.starts, sq.lens)], sq.page)
    g = torch.Generator(device=gpu).manual_seed(seed)
    kv = [torch.randn(whole.tokens, heads, dim, generator=g, device=gpu) * s for s in scale]
    ck.kv_write(cache, ck.KvBatch(batch.page_table, _i32(whole.starts, gpu), _i32(whole.offsets, gpu), whole.tokens), *kv)


@pytest.mark.parametrize("typ,heads,dim,page,order", [
    ("bf16", 8, 128, 64, "phsd"), ("f16", 3, 96, 16, "pshd"), ("f32", 1, 32, 32, "hpsd"), ("bf16", 5, 256, 16, "phsd"),
    ("f32", 2, 224, 128, "pshd"), ("f16", 7, 64, 256, "sphd")])
def test_write_and_read(gpu, typ, heads, dim, page, order):
    print(f"[case] write/read {typ} heads={heads} dim={dim} page={page} {order}", flush=True)
    sq = ko.Seqs([5, 0, 130, 17, 0], [1, 33, 0, 100, 257], page, seed=dim)
    sq.table[3, 0] = -1 if page > 16 else sq.table[3, 0]     # an unmapped page (its tokens are not stored)
    sq.table[4, 1 if page <= 128 else 0] = sq.n_pages + 5 if page != 256 else sq.table[4, 0]
    cache = _cache(sq, heads, dim, gpu, order)
    before = [_bytes(t).clone() for t in cache.tensors()]
    b = _batch(sq, gpu)
    g = torch.Generator().manual_seed(dim)
    x = [torch.randn(sq.tokens, heads, dim, generator=g) * torch.exp(3 * torch.randn(sq.tokens, heads, 1, generator=g)) for _ in range(2)]
    x[0][7] = 0                       # an empty row, a tiny one, an infinite group, one with NaN
    x[0][8] *= 0 if typ == "f16" else 1e-36
    x[1][9, 0, 3] = float("inf")
    x[1][10, heads - 1, dim - 1] = float("nan")
    x[1][11, 0, :32] = torch.tensor([7.0, 5, 3.5, 2.5, 1.75, 1.25, .75, .25] * 4) * torch.tensor([1.0, -1] * 16)  # ties, the largest at the border
    x[1][12, 0, :32] = x[1][11, 0, :32] * 2 ** -6
    x[1][12, 0, 0] = 7.03125 * 2 ** -6  # past the border: the next power
    x = [t.to(TYPES[typ]) for t in x]
    if typ != "f16":
        x[0][13] = torch.finfo(torch.float32).max if typ == "f32" else torch.finfo(torch.bfloat16).max
        x[0][14] *= 2.0 ** -98
    ck.kv_write(cache, b, *(t.to(gpu) for t in x))
    out = tuple(torch.full((sq.tokens, heads, dim), 7.0, dtype=TYPES[typ], device=gpu) for _ in range(2))
    ck.kv_read(cache, b, TAGS[typ], out=out)
    torch.cuda.synchronize()
    touched = torch.zeros(sq.n_pages, sq.page, dtype=torch.bool)
    for which, name in enumerate(("k", "v")):
        got, got_s = k4.unpack(_bytes(getattr(cache, name)).cpu()), _bytes(getattr(cache, name + "_scale")).cpu()
        codes, byte = k4.quantise(x[which].float())
        power = torch.where(byte == 255, torch.tensor(float("nan"), dtype=torch.float64), torch.exp2(byte.double() - 127))
        back = (codes * power.repeat_interleave(32, -1)).to(TYPES[typ])
        t = 0
        for s in range(len(sq.lens)):
            for i in range(sq.lens[s]):
                p, slot = sq.place(s, sq.starts[s] + i)
                if p < 0:
                    assert (out[which][t] == 0).all(), (s, i)
                else:
                    touched[p, slot] = True
                    assert torch.equal(got_s[p, :, :, slot], byte[t]), (s, i, got_s[p, :, :, slot], byte[t])
                    assert torch.equal(got[p, :, slot], codes[t]), (s, i)
                    assert torch.equal(torch.nan_to_num(out[which][t].cpu().double(), nan=5e4), torch.nan_to_num(back[t].double(), nan=5e4)), (s, i)
                t += 1
    for old, new in zip(before, cache.tensors()):   # nothing else was written
        a, c = old, _bytes(new)
        if a.shape[2:] == (dim // 32, sq.page):
            a, c = a.transpose(2, 3), c.transpose(2, 3)
        a, c = (z.transpose(1, 2)[~touched.to(gpu)] for z in (a, c))
        assert torch.equal(a, c)


ATTEND = [
    # q type, kv heads, group, dim, page, starts, lens, window
    ("bf16", 8, 4, 128, 64, [1000], [1], 0),
    ("bf16", 2, 4, 128, 16, [0, 5, 63, 64, 700], [1, 1, 1, 1, 1], 0),
    ("f16", 1, 8, 64, 32, [31, 32, 200], [1, 2, 1], 0),
    ("bf16", 2, 1, 128, 128, [100, 0], [1, 1], 50),
    ("f16", 3, 2, 96, 16, [250, 0, 9], [1, 1, 5], 0),
    ("bf16", 1, 16, 256, 64, [129], [1], 0),
    ("f16", 1, 4, 224, 16, [129, 3], [1, 4], 0),
    ("bf16", 1, 20, 32, 16, [77, 300], [1, 1], 0),
    ("bf16", 2, 4, 128, 64, [0], [300], 0),
    ("bf16", 1, 4, 128, 32, [190, 0, 64], [70, 130, 1], 0),
    ("f16", 1, 8, 128, 16, [0, 33], [150, 64], 0),
    ("bf16", 2, 2, 64, 256, [500], [65], 0),
    ("f16", 2, 3, 96, 64, [40, 0], [129, 31], 33),
    ("bf16", 1, 2, 256, 16, [90], [100], 0),
    ("f16", 1, 1, 32, 16, [10, 0], [40, 200], 64),
    ("bf16", 1, 7, 64, 16, [3, 0, 0, 400], [17, 0, 1, 9], 10),
    ("f16", 1, 4, 256, 32, [70, 0], [40, 90], 0),
    ("bf16", 1, 5, 160, 16, [2000], [3], 0),
    ("bf16", 1, 8, 64, 64, [1500], [40], 0),
    ("f16", 1, 4, 32, 128, [700], [80], 0),
]


def _attend(gpu, typ, heads, group, dim, page, starts, lens, window, sq=None, scale=None, order="phsd", loud=1.0, change=None):
    sq = sq or ko.Seqs(starts, lens, page, seed=len(starts))
    cache = _cache(sq, heads, dim, gpu, order)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, heads, dim, gpu, 3)
    if change:
        change(sq, cache)
    g = torch.Generator(device=gpu).manual_seed(4)
    q = (torch.randn(sq.tokens, heads * group, dim, generator=g, device=gpu) * loud).to(TYPES[typ])
    plan = ck.KvAttention(heads * group, heads, dim, len(starts), sq.tokens, max(lens), max(o + n for o, n in zip(starts, lens)))
    out = torch.full_like(q, 9.0)
    lse = torch.full((sq.tokens, heads * group), 9.0, device=gpu)
    plan.run(cache, b, q, scale=scale, window=window, out=out, lse=lse)
    torch.cuda.synchronize()
    return sq, cache, b, q, plan, out, lse


def _check(sq, cache, q, out, lse, group, window, scale=None):
    D = q.shape[2]
    k, v = (k4.as_numpy(_values(cache, n)) for n in ("k", "v"))
    ref = ko.attention(sq, k, v, q.cpu().double().numpy(), group, D ** -0.5 if scale is None else scale, window)
    # scores are sums of 2 D exact products (float16 queries may come in two halves); weights
    # have 11 bits at least, their smallest step 2^-32 of the largest
    bound, lbound = ko.attention_bounds(*ref, 2 * D, 2.0 ** -11, q.dtype, np.abs(v).max())
    err = np.abs(out.cpu().double().numpy() - ref[0])
    print(f"  largest error / bound: {(err / bound).max():.3f}", flush=True)
    assert (err <= bound).all()
    got, none = lse.cpu().double().numpy(), ~np.isfinite(ref[1])
    assert (got[none] == -np.inf).all()
    assert (np.abs(got[~none] - ref[1][~none]) <= np.broadcast_to(lbound, got.shape)[~none]).all()


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "-".join(map(str, c[:5])))
def test_attention(gpu, case):
    print(f"[case] attend {case}", flush=True)
    typ, heads, group, dim, page, starts, lens, window = case
    sq, cache, b, q, plan, out, lse = _attend(gpu, *case)
    _check(sq, cache, q, out, lse, group, window)
    # the same call again on the same workspace, and without hints or lse
    again = torch.full_like(q, 5.0)
    plan.run(cache, b, q, window=window, out=again)
    torch.cuda.synchronize()
    assert torch.equal(again, out)
    plan2 = ck.KvAttention(heads * group, heads, dim, len(starts), sq.tokens)
    loose = plan2.run(cache, _batch(sq, gpu, hints=False), q, window=window)
    _check(sq, cache, q, loose, lse, group, window)


@pytest.mark.parametrize("typ,dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 90, 2], [200, 100, 7]])
def test_unmapped_pages_and_rows_without_keys(gpu, typ, dim, lens):
    """Evicted pages are not attended to; rows that see none give zeros and -inf; what
    lies in masked places (powers of NaN everywhere here) never shows."""
    print(f"[case] unmapped {typ} {dim} {lens}", flush=True)
    starts = [100, 20, 300]
    sq = ko.Seqs(starts, lens, 16, seed=8)
    full = sq.table.copy()
    cache = _cache(sq, 2, dim, gpu)
    _fill(sq, cache, _batch(sq, gpu), 2, dim, gpu, 3)
    sq.table[0, :4] = [-1, -7, sq.n_pages, 2**31 - 1]
    sq.table[1, :] = -1                      # nothing left of sequence 1
    sq.table[2, 3:17] = -1
    for s, c in ((0, 0), (0, 1), (2, 5)):    # poison the pages that went away
        _bytes(cache.k_scale)[int(full[s, c])] = 255
        _bytes(cache.v_scale)[int(full[s, c])] = 255
    g = torch.Generator(device=gpu).manual_seed(4)
    q = torch.randn(sq.tokens, 8, dim, generator=g, device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(8, 2, dim, 3, sq.tokens, max(lens), 500)
    for window in (0, 30):
        lse = torch.full((sq.tokens, 8), 9.0, device=gpu)
        out = plan.run(cache, _batch(sq, gpu), q, window=window, lse=lse)
        torch.cuda.synchronize()
        assert (out[lens[0]:lens[0] + lens[1]] == 0).all()
        _check(sq, cache, q, out, lse, 4, window)
    sq.table = sq.table[:, :2].copy()        # a table narrower than the contexts
    lse = torch.full((sq.tokens, 8), 9.0, device=gpu)
    out = plan.run(cache, _batch(sq, gpu), q, lse=lse)
    torch.cuda.synchronize()
    _check(sq, cache, q, out, lse, 4, 0)


@pytest.mark.parametrize("typ,dim,lens,group", [("bf16", 128, [1], 4), ("f16", 96, [1], 4), ("bf16", 64, [3], 2), ("bf16", 256, [2], 4),
                                                ("f16", 128, [20], 4), ("bf16", 64, [30], 4), ("bf16", 256, [40], 4),
                                                ("bf16", 128, [90], 4), ("f16", 64, [80], 4)])
def test_groups_of_nan_reach_who_sees_them_only(gpu, typ, dim, lens, group):
    """A key's group of NaN makes every token that sees it NaN; a value's its 32 dimensions
    alone, and leaves the log-sum; a token whose window ends after it neither."""
    print(f"[case] NaN {typ} {dim} {lens}", flush=True)
    sq = ko.Seqs([200], lens, 16, seed=1)
    cache = _cache(sq, 2, dim, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, dim, gpu, 3)
    p, slot = sq.place(0, 100)
    q = torch.randn(sq.tokens, 2 * group, dim, device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(2 * group, 2, dim, 1, sq.tokens, max(lens), 400)
    lse = [torch.empty(sq.tokens, 2 * group, device=gpu) for _ in range(2)]
    want = plan.run(cache, b, q, lse=lse[0])
    far = plan.run(cache, b, q, window=100)
    last = dim // 32 - 1
    keep = int(_bytes(cache.v_scale)[p, 1, last, slot])
    _bytes(cache.v_scale)[p, 1, last, slot] = 255
    got = plan.run(cache, b, q, lse=lse[1])
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[:, group:, 32 * last:] = True
    assert torch.equal(torch.isnan(got), bad) and torch.equal(lse[0], lse[1])
    # the other values: nothing but which power float16 values are held against may differ
    assert (got[~bad].float() - want[~bad].float()).abs().max() <= 2 * ko.UNIT[q.dtype] * want.float().abs().max()
    assert torch.equal(plan.run(cache, b, q, window=100), far)
    # seen by some rows of a tile only: the window of the first tokens holds it
    if lens[0] > 1:
        some = plan.run(cache, b, q, window=101 + lens[0] // 2)   # position 200 + i sees 100 up to i = lens // 2
        rows = torch.isnan(some[:, group:, 32 * last:]).all(-1).all(-1).cpu()
        assert torch.equal(rows, torch.arange(sq.tokens) <= lens[0] // 2)
        assert not torch.isnan(some[lens[0] // 2 + 1:]).any() and not torch.isnan(some[:, :group]).any()
    _bytes(cache.v_scale)[p, 1, last, slot] = keep
    _bytes(cache.k_scale)[p, 0, 0, slot] = 255
    got = plan.run(cache, b, q)
    assert torch.isnan(got[:, :group]).all() and torch.equal(got[:, group:], want[:, group:])
    assert torch.equal(plan.run(cache, b, q, window=100), far)


@pytest.mark.parametrize("typ,dim,lens,group", [("bf16", 128, [1], 4), ("f16", 128, [2], 4), ("bf16", 128, [25], 4), ("f16", 64, [30], 4),
                                                ("f16", 256, [40], 2), ("bf16", 256, [40], 2), ("bf16", 128, [100], 4), ("f16", 128, [100], 4),
                                                ("bf16", 64, [100], 4)])
@pytest.mark.parametrize("up", [20, -20, 90])
def test_scales_far_apart(gpu, typ, dim, lens, group, up):
    """Later keys' values 2^up times the first ones' in one group of dimensions (up to what
    float16 does not hold beside the first: a block begins again), and for |up| = 20 keys so too."""
    if typ == "f16" and up == 90:
        pytest.skip("outputs of float16 end at 65504")
    print(f"[case] far apart {typ} {dim} {lens} {up}", flush=True)

    def change(sq, cache):
        last = dim // 32 - 1
        for j in range(250, 300):
            p, slot = sq.place(0, j)
            _bytes(cache.v_scale)[p, :, last, slot] += up if up > 0 else 0
            if abs(up) == 20:
                _bytes(cache.k_scale)[p, :, last, slot] -= 20
        for j in range(0, 200):
            p, slot = sq.place(0, j)
            _bytes(cache.v_scale)[p, :, last, slot] -= -up if up < 0 else 0
        if typ == "f16" and up > 0:                                     # outputs within float16
            _bytes(cache.v_scale)[:, :, last] -= 10

    sq, cache, b, q, plan, out, lse = _attend(gpu, typ, 2, group, dim, 16, [400], lens, 0, change=change)
    D, (k, v) = dim, (k4.as_numpy(_values(cache, n)) for n in ("k", "v"))
    ref = ko.attention(sq, k, v, q.cpu().double().numpy(), group, D ** -0.5, 0)
    n_groups = dim // 32
    for g in range(n_groups):   # each group of dimensions against its own largest value
        part = slice(32 * g, 32 * g + 32)
        bound, lbound = ko.attention_bounds(ref[0][..., part], ref[1], ref[2][..., part], ref[3], ref[4], 2 * D, 2.0 ** -11, q.dtype, np.abs(v[..., part]).max())
        # values below 2^-23 of the largest scale are off by 2^-25 of that
        bound = bound + 2.0 ** -25 * np.abs(v[..., part]).max()
        err = np.abs(out.cpu().double().numpy()[..., part] - ref[0][..., part])
        assert (err <= bound).all(), g
    assert (np.abs(lse.cpu().double().numpy() - ref[1]) <= np.broadcast_to(lbound, ref[1].shape)).all()


@pytest.mark.parametrize("lens", [[1], [60], [120]])
@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_keys_later_than_a_block_expects(gpu, lens, typ):
    """Later keys 2^20 times the first ones', as float16 does not hold them against the first."""
    def change(sq, cache):
        for j in range(0, 300):
            p, slot = sq.place(0, j)
            _bytes(cache.k_scale)[p, :, :, slot] -= 20
        _bytes(cache.v_scale)[:] += 3
    sq, cache, b, q, plan, out, lse = _attend(gpu, typ, 1, 4, 128, 32, [400], lens, 0, change=change)
    _check(sq, cache, q, out, lse, 4, 0)


@pytest.mark.parametrize("typ,dim,lens", [("bf16", 128, [40]), ("f16", 256, [40]), ("bf16", 64, [100]), ("f16", 128, [100]), ("bf16", 128, [1])])
@pytest.mark.parametrize("first", ["unmapped", "zeros"])
@pytest.mark.parametrize("power", [0, -60, 60])
def test_first_keys_without_a_scale(gpu, typ, dim, lens, first, power):
    """A block whose first keys are not mapped, or zeros, has no scale to begin with; those after may be of any size."""
    if typ == "f16" and power > 0:
        pytest.skip("outputs of float16 end at 65504")
    print(f"[case] first keys {typ} {dim} {lens} {first} {power}", flush=True)
    sq = ko.Seqs([600], lens, 16, seed=2)

    def change(sq, cache):
        for t in (cache.k_scale, cache.v_scale):
            _bytes(t)[:] += power if power > 0 else 0
            _bytes(t)[:] -= -power if power < 0 else 0
        if typ == "f16" or power > 0:
            _bytes(cache.k_scale)[:] -= power if power > 0 else 0
            _bytes(cache.k_scale)[:] += -power if power < 0 else 0
        if first == "zeros":
            for j in range(230):
                p, slot = sq.place(0, j)
                for t in (cache.k, cache.v):
                    _bytes(t)[p, :, slot] = 0
                for t in (cache.k_scale, cache.v_scale):
                    _bytes(t)[p, :, :, slot] = 0

    if first == "zeros":
        sq, cache, b, q, plan, out, lse = _attend(gpu, typ, 2, 4, dim, 16, [600], lens, 0, sq=sq, change=change)
    else:
        cache = _cache(sq, 2, dim, gpu)
        _fill(sq, cache, _batch(sq, gpu), 2, dim, gpu, 3)
        change(sq, cache)
        sq.table[0, :14] = -1
        q = torch.randn(sq.tokens, 8, dim, device=gpu).to(TYPES[typ])
        lse = torch.full((sq.tokens, 8), 9.0, device=gpu)
        out = ck.KvAttention(8, 2, dim, 1, sq.tokens, max(lens), 700).run(cache, _batch(sq, gpu), q, lse=lse)
        torch.cuda.synchronize()
    if typ == "f16" and power < 0:      # outputs of 2^-60 are 0 in float16
        assert out.abs().max() < 2.0 ** -24
        return
    D, (k, v) = dim, (k4.as_numpy(_values(cache, n)) for n in ("k", "v"))
    ref = ko.attention(sq, k, v, q.cpu().double().numpy(), 4, D ** -0.5, 0)
    bound, lbound = ko.attention_bounds(*ref, 2 * D, 2.0 ** -11, q.dtype, np.abs(v).max())
    bound = bound - 2.0 ** -24 + 2.0 ** -24 * np.abs(v).max()   # the bound's absolute part, at the values' size
    err = np.abs(out.cpu().double().numpy() - ref[0])
    assert (err <= bound).all(), (err / bound).max()
    assert (np.abs(lse.cpu().double().numpy() - ref[1]) <= np.broadcast_to(lbound, ref[1].shape)).all()


@pytest.mark.parametrize("lens", [[1, 2], [70, 8]])
@pytest.mark.parametrize("loud,scale", [(40.0, None), (0.0, None), (1.0, 0.0), (1.0, -0.3)])
def test_peaked_and_flat_scores(gpu, lens, loud, scale):
    sq, cache, b, q, plan, out, lse = _attend(gpu, "bf16", 2, 4, 128, 64, [500, 30], lens, 0, loud=loud, scale=scale)
    _check(sq, cache, q, out, lse, 4, 0, scale)


@pytest.mark.parametrize("n", [1, 37, 150])
def test_strides_and_orders(gpu, n):
    """Caches in every order of axes, queries and outputs as slices of wider tensors."""
    for order in ("pshd", "hpsd", "sphd"):
        sq, cache, b, q, plan, out, lse = _attend(gpu, "bf16", 2, 2, 64, 16, [90, 7], [n, 3], 0, order=order)
        _check(sq, cache, q, out, lse, 2, 0)
        wide = torch.zeros(sq.tokens, 9, 128, dtype=torch.bfloat16, device=gpu)
        wide[:, 2:6, 32:96] = q
        to = torch.full((sq.tokens, 7, 64), 3.0, dtype=torch.bfloat16, device=gpu)
        plan.run(cache, b, wide[:, 2:6, 32:96], out=to[:, 1:5])
        torch.cuda.synchronize()
        assert torch.equal(to[:, 1:5], out) and (to[:, 0] == 3).all() and (to[:, 5:] == 3).all()


def test_offsets_past_32_bits(gpu):
    """Pages further apart than 2^32 bytes, of codes and of powers."""
    far = (1 << 32) + 4096
    raw = [torch.zeros(far + (1 << 20), dtype=torch.uint8, device=gpu) for _ in range(4)]
    k, v = (r.as_strided((2, 1, 16, 64), (far, 16 * 64, 64, 1)).view(torch.float4_e2m1fn_x2) for r in raw[:2])
    ks, vs = (r.as_strided((2, 1, 4, 16), (far, 64, 16, 1)).view(torch.float8_e8m0fnu) for r in raw[2:])
    cache = ck.KvCache(k, v, ks, vs)
    sq = ko.Seqs([0], [32], 16, spare=0)
    sq.table[0] = [1, 0]
    b = _batch(sq, gpu)
    g = torch.Generator(device=gpu).manual_seed(2)
    x = [torch.randn(32, 1, 128, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2)]
    ck.kv_write(cache, b, *x)
    near = ck.KvCache.empty(2, 16, 1, 128, ck.F4)
    ck.kv_write(near, b, *x)
    for a, c in zip(ck.kv_read(cache, b), ck.kv_read(near, b)):
        assert torch.equal(a, c)
    plan = ck.KvAttention(4, 1, 128, 1, 32)
    for n in (1, 16, 32):       # few and many rows
        bb = ck.KvBatch(b.page_table, _i32([32 - n], gpu), _i32([0, n], gpu), n)
        q = torch.randn(n, 4, 128, generator=g, device=gpu).to(torch.bfloat16)
        assert torch.equal(plan.run(cache, bb, q), plan.run(near, bb, q))


def test_another_stream_and_a_graph(gpu):
    """Write, read and attention on a side stream, then captured: every replay (with eager
    work and synchronisation between) equals the eager result."""
    sq = ko.Seqs([300, 40], [1, 1], 16, seed=5)
    cache = _cache(sq, 2, 128, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 128, gpu, 3)
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


def test_one_workspace_for_caches_of_several_types(gpu):
    """A plan runs 4- and 8-bit caches and every kernel in turn."""
    sq = ko.Seqs([700, 20], [1, 1], 16, seed=3)
    four, eight = _cache(sq, 2, 128, gpu), ck.KvCache.empty(sq.n_pages, 16, 2, 128, ck.F8)
    b = _batch(sq, gpu)
    for c in (four, eight):
        _fill(sq, c, b, 2, 128, gpu, 3)
    plan = ck.KvAttention(8, 2, 128, 2, 200, 100, 900)
    q = torch.randn(200, 8, 128, device=gpu).to(torch.bfloat16)
    chunks = [([700, 20], [1, 1]), ([650, 0], [20, 10]), ([600, 0], [100, 20])]
    first = {}
    for turn in range(2):
        for i, (starts, lens) in enumerate(chunks):
            bb = ck.KvBatch(b.page_table, _i32(starts, gpu), _i32(np.concatenate([[0], np.cumsum(lens)]), gpu), sum(lens), max(lens), 701)
            for name, c in (("four", four), ("eight", eight)):
                got = plan.run(c, bb, q[:sum(lens)])
                if turn:
                    assert torch.equal(first[i, name], got)
                first[i, name] = got


def test_empty_batches(gpu):
    cache = ck.KvCache.empty(2, 16, 1, 64, ck.F4)
    b = ck.KvBatch(_i32([[0]], gpu), _i32([0], gpu), _i32([0, 0], gpu), 0)
    none = torch.zeros(0, 1, 64, dtype=torch.bfloat16, device=gpu)
    ck.kv_write(cache, b, none, none)
    assert all(t.shape == (0, 1, 64) for t in ck.kv_read(cache, b))
    assert ck.KvAttention(1, 1, 64, 1, 1).run(cache, b, none).shape == (0, 1, 64)


def test_refusals(gpu):
    def bad(part, f, *a, **kw):
        with pytest.raises(ck.CkrError) as e:
            f(*a, **kw)
        assert e.value.code == ck.CKR_E_INVALID and part in str(e.value), str(e.value)

    cache = ck.KvCache.empty(3, 16, 2, 64, ck.F4)
    k, v, ks, vs = cache.tensors()
    assert k.shape == (3, 2, 16, 32) and ks.shape == (3, 2, 2, 16) and cache.head_dim == 64
    bad("scales belong", ck.KvCache, k, v)
    bad("scales must be", ck.KvCache, k, v, torch.zeros(3, 2, 16, device=gpu), torch.zeros(3, 2, 16, device=gpu))
    bad("scales must be", ck.KvCache, k, v, ks.view(torch.uint8), vs.view(torch.uint8))
    bad("scales must be", ck.KvCache, k, v, ks.view(3, 2, 16, 2), vs.view(3, 2, 16, 2))
    bad("multiple of 32", ck.KvCache.empty, 3, 16, 2, 80, ck.F4)
    half = torch.zeros(3, 2, 16, 24, dtype=torch.uint8, device=gpu).view(torch.float4_e2m1fn_x2)
    bad("multiple of 32", ck.KvCache, half, half, ks, vs)
    b = ck.KvBatch(_i32([[0, 1, 2]], gpu), _i32([10], gpu), _i32([0, 2], gpu), 2)
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=gpu)
    bad("[2, 2, 64]", ck.kv_write, cache, b, x[..., :32], x)
    bad("not dtype", ck.kv_read, cache, b, ck.F4)
    flat = torch.zeros(3 * 2 * 16 * 32 + 8, dtype=torch.uint8, device=gpu)
    odd = flat[8:].view(3, 2, 16, 32).view(torch.float4_e2m1fn_x2)
    bad("16-byte", ck.kv_write, ck.KvCache(odd, v, ks, vs), b, x, x)
    near = torch.zeros(3, 2, 16, 40, dtype=torch.uint8, device=gpu)[..., :32].view(torch.float4_e2m1fn_x2)
    bad("multiples of 16 bytes", ck.kv_write, ck.KvCache(near, near, ks, vs), b, x, x)
    same = k[:1].view(torch.uint8).expand(3, 2, 16, 32).view(torch.float4_e2m1fn_x2)
    bad("overlap", ck.kv_write, ck.KvCache(same, v, ks, vs), b, x, x)
    scales = ks[:1].view(torch.uint8).expand(3, 2, 2, 16).view(torch.float8_e8m0fnu)
    bad("overlap", ck.kv_write, ck.KvCache(k, v, scales, vs), b, x, x)
    bad("8-bit floats or int8", ck.add_rms_norm, x[0], None, torch.ones(64, dtype=torch.bfloat16, device=gpu), dtype=ck.F4)
    torch.cuda.synchronize()
