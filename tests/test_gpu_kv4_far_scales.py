"""Attention over a cache in 4 bits whose scales are further apart than 16 bits hold side by
side: what a row gets depends on the keys that it sees, not on others of its tile, and not on
the hints that choose the kernel.  Bounds of each row from what it sees itself."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests import kv4_oracle as k4
from tests import kv_oracle as ko
from tests.test_gpu_kv4 import TYPES, _batch, _bytes, _cache, _fill, _i32, _values

pytestmark = pytest.mark.gpu


def _seen_most(sq, v, group, heads, window):
    """Of each row, the largest magnitude among the values that it sees, by groups of 32."""
    most = np.zeros((sq.tokens, heads * group, v.shape[-1]))
    g = np.abs(v).reshape(*v.shape[:-1], -1, 32).max(-1).repeat(32, -1)
    for s, (o, n) in enumerate(zip(sq.starts, sq.lens)):
        for i in range(n):
            for j in range(max(0, o + i + 1 - window) if window else 0, o + i + 1):
                p, slot = sq.place(s, j)
                if p >= 0:
                    t = int(sq.offsets[s]) + i
                    most[t] = np.maximum(most[t], g[p, :, slot].repeat(group, 0))
    return most


def _check_rows(sq, cache, q, out, lse, group, window):
    k, v = (k4.as_numpy(_values(cache, n)) for n in ("k", "v"))
    ref = ko.attention(sq, k, v, q.cpu().double().numpy(), group, q.shape[2] ** -0.5, window)
    most = _seen_most(sq, v, group, cache.n_heads, window)
    # weights have 11 bits, their smallest step is 2^-32 of the largest: of the values that the row sees
    bound, lbound = ko.attention_bounds(*ref, 2 * q.shape[2], 2.0 ** -11, q.dtype, 0.0)
    bound = bound + ref[4][:, None, None] * most * 2.0 ** -32
    bound = bound - 2.0 ** -24 + (2.0 ** -24 if q.dtype == torch.float16 else 2.0 ** -100)
    err = np.abs(out.cpu().double().numpy() - ref[0])
    worst = np.unravel_index((err / bound).argmax(), err.shape)
    assert (err <= bound).all(), (worst, err[worst] / bound[worst], ref[0][worst])
    none = ~np.isfinite(ref[1])
    got = lse.cpu().double().numpy()
    assert (got[none] == -np.inf).all()
    assert (np.abs(got - ref[1])[~none] <= np.broadcast_to(lbound, got.shape)[~none]).all()


def _shift(sq, cache, which, keys, by, groups=slice(None)):
    for j in keys:
        p, slot = sq.place(0, j)
        t = _bytes(getattr(cache, which + "_scale"))
        t[p, :, groups, slot] = (t[p, :, groups, slot].int() + by).clamp(1, 252).to(torch.uint8)


CASES = [
    # q type, heads, group, dim, page, old tokens, chunk, window, max_context given
    ("bf16", 2, 4, 128, 16, 0, 30, 0, None),      # 120 rows a head
    ("f16", 2, 4, 128, 64, 70, 30, 0, None),
    ("bf16", 1, 2, 64, 32, 200, 64, 0, None),
    ("f16", 1, 4, 64, 16, 0, 32, 20, None),
    ("bf16", 1, 2, 256, 16, 100, 60, 0, None),
    ("f16", 1, 1, 224, 16, 0, 100, 0, None),
    ("bf16", 2, 4, 128, 64, 0, 90, 0, None),       # 360
    ("f16", 1, 8, 128, 16, 300, 40, 0, None),
    ("bf16", 1, 4, 96, 16, 0, 150, 40, None),
    ("f16", 2, 3, 64, 128, 0, 130, 0, None),
    ("bf16", 1, 4, 128, 32, 90, 70, 0, 100),       # one split
    ("f16", 1, 4, 32, 16, 0, 100, 0, 60),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("how", ["late values", "early values", "late keys", "one group", "as far as held"])
def test_rows_keep_what_they_see(gpu, case, how):
    typ, heads, group, dim, page, old, chunk, window, context = case
    print(f"[case] {how} {case}", flush=True)
    sq = ko.Seqs([old], [chunk], page, seed=chunk)
    cache = _cache(sq, heads, dim, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, heads, dim, gpu, 3)
    border, end = old + chunk // 2, old + chunk
    up, down = (13, 13) if typ == "f16" else (40, 0)        # outputs of float16 end at 65504
    if how == "late values":
        _shift(sq, cache, "v", range(0, border), -down)
        _shift(sq, cache, "v", range(border, end), up)
    elif how == "early values":                              # rows in the end see the small ones only where a window hides the rest
        _shift(sq, cache, "v", range(0, border), up)
        _shift(sq, cache, "v", range(border, end), -down)
    elif how == "late keys":
        _shift(sq, cache, "k", range(border, end), 28)
    elif how == "as far as held":                            # 20 octaves, and a few between groups of one size
        _shift(sq, cache, "v", range(0, border), -10)
        _shift(sq, cache, "v", range(border, end), 10)
        _shift(sq, cache, "k", range(0, border), -20)
    else:
        _shift(sq, cache, "v", range(border, end, 2), up, slice(0, 1))
        _shift(sq, cache, "v", range(0, border), -down, slice(0, 1))
    if context is not None:
        b = ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, chunk, context)
    q = torch.randn(sq.tokens, heads * group, dim, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(heads * group, heads, dim, 1, sq.tokens, chunk, old + chunk)
    lse = torch.full((sq.tokens, heads * group), 9.0, device=gpu)
    out = plan.run(cache, b, q, window=window, lse=lse)
    again = plan.run(cache, b, q, window=window)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    _check_rows(sq, cache, q, out, lse, group, window)


@pytest.mark.parametrize("typ,group,chunk", [("bf16", 4, 30), ("f16", 4, 30), ("bf16", 4, 90), ("f16", 4, 90)])
def test_far_scales_beside_nan_and_unmapped_pages(gpu, typ, group, chunk):
    """A value's group of NaN, a key's, and pages that are not mapped, in such blocks: the same
    as of the kernel that the hint of single tokens chooses."""
    print(f"[case] NaN and gaps {typ} {group} {chunk}", flush=True)
    sq = ko.Seqs([100], [chunk], 16, seed=2)
    cache = _cache(sq, 2, 128, gpu)
    _fill(sq, cache, _batch(sq, gpu), 2, 128, gpu, 3)
    _shift(sq, cache, "v", range(0, 100 + chunk // 2), -13)
    _shift(sq, cache, "v", range(100 + chunk // 2, 100 + chunk), 13)
    p, slot = sq.place(0, 100 + chunk // 3)
    _bytes(cache.v_scale)[p, 1, 2, slot] = 255
    p, slot = sq.place(0, 100 + chunk - 2)
    _bytes(cache.k_scale)[p, 0, 0, slot] = 255
    sq.table[0, 1:3] = -1
    b = _batch(sq, gpu)
    few = ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, 1, 100 + chunk)
    q = torch.randn(sq.tokens, 2 * group, 128, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(2 * group, 2, 128, 1, sq.tokens, chunk, 100 + chunk)
    for window in (0, 45):
        lse = [torch.full((sq.tokens, 2 * group), 9.0, device=gpu) for _ in range(2)]
        out, want = (plan.run(cache, x, q, window=window, lse=y) for x, y in ((b, lse[0]), (few, lse[1])))
        torch.cuda.synchronize()
        assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(torch.isnan(lse[0]), torch.isnan(lse[1]))
        assert torch.isnan(out).any() and not torch.isnan(out).all()
        ok = ~torch.isnan(want)
        # two roundings of sums that differ by what 11 bits of the weights and of a value's 16 make; float16 below
        # 2^-14 (first tokens' values are 2^-13 times normal ones) has steps of 2^-24, of which either is off by a half
        out, want = (torch.nan_to_num(x.float(), nan=0.0) for x in (out, want))
        assert ((out - want).abs()[ok] <= (2 * ko.UNIT[q.dtype] * want.abs() + 2.0 ** -10 * want.abs().amax(-1, keepdim=True) + 2.0 ** -24 * (typ == "f16"))[ok]).all()


def test_groups_without_values_are_no_scales(gpu):
    """Zeros (byte 0) beside large values: the usual kernels' results, bit for bit as with other zeros."""
    sq = ko.Seqs([60], [90], 16, seed=1)
    cache = _cache(sq, 1, 128, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 1, 128, gpu, 3)
    for j in range(0, 150, 3):
        p, slot = sq.place(0, j)
        _bytes(cache.v)[p, :, slot] = 0
        _bytes(cache.v_scale)[p, :, :, slot] = 120
    q = torch.randn(90, 4, 128, device=gpu).to(torch.bfloat16)
    plan = ck.KvAttention(4, 1, 128, 1, 90, 90, 150)
    want = plan.run(cache, b, q)
    for j in range(0, 150, 3):
        p, slot = sq.place(0, j)
        _bytes(cache.v_scale)[p, :, :, slot] = 0
    assert torch.equal(plan.run(cache, b, q), want)


@pytest.mark.parametrize("typ,lens,window", [("bf16", [40, 3, 25, 0, 30], 0), ("f16", [30, 90, 1], 0), ("bf16", [70, 90], 60)])
def test_several_sequences(gpu, typ, lens, window):
    """Far scales in one sequence, on pages of its own, beside others without."""
    print(f"[case] several {typ} {lens} {window}", flush=True)
    starts = [60, 200, 17, 5, 130][:len(lens)]
    sq = ko.Seqs(starts, lens, 16, seed=4)
    cache = _cache(sq, 2, 128, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 128, gpu, 3)
    _shift(sq, cache, "v", range(0, starts[0] + lens[0] // 2), -13)
    _shift(sq, cache, "v", range(starts[0] + lens[0] // 2, starts[0] + lens[0]), 13)
    q = torch.randn(sq.tokens, 8, 128, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(8, 2, 128, len(lens), sq.tokens, max(lens), 300)
    lse = torch.full((sq.tokens, 8), 9.0, device=gpu)
    out = plan.run(cache, b, q, window=window, lse=lse)
    torch.cuda.synchronize()
    _check_rows(sq, cache, q, out, lse, 4, window)


@pytest.mark.parametrize("typ", ["bf16", "f16"])
def test_slots_far_apart(gpu, typ):
    """Slots of a page 2^26 bytes apart, which the 128-row kernel alone takes: near and far scales."""
    step, page = 1 << 26, 16
    raw = [torch.zeros((page - 1) * step + 64, dtype=torch.uint8, device=gpu) for _ in range(2)]
    k, v = (r.as_strided((1, 1, page, 64), (0, 0, step, 1)).view(torch.float4_e2m1fn_x2) for r in raw)
    ks, vs = (torch.zeros(1, 1, 4, page, dtype=torch.uint8, device=gpu).view(torch.float8_e8m0fnu) for _ in range(2))
    cache = ck.KvCache(k, v, ks, vs)
    sq = ko.Seqs([0], [page], page, spare=0)
    b = _batch(sq, gpu)
    g = torch.Generator(device=gpu).manual_seed(2)
    ck.kv_write(cache, b, *(torch.randn(page, 1, 128, generator=g, device=gpu) for _ in range(2)))
    q = torch.randn(page, 12, 128, generator=g, device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(12, 1, 128, 1, page, page, page)
    for far in (False, True):
        if far:
            _shift(sq, cache, "v", range(0, 8), -13)
            _shift(sq, cache, "v", range(8, 16), 13)
        lse = torch.full((page, 12), 9.0, device=gpu)
        out = plan.run(cache, b, q, lse=lse)
        torch.cuda.synchronize()
        _check_rows(sq, cache, q, out, lse, 12, 0)


@pytest.mark.parametrize("typ,chunk", [("bf16", 30), ("f16", 90)])
def test_captured(gpu, typ, chunk):
    """A captured call whose scales move apart and together between replays."""
    sq = ko.Seqs([100], [chunk], 16, seed=2)
    cache = _cache(sq, 2, 128, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, 2, 128, gpu, 3)
    q = torch.randn(sq.tokens, 8, 128, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(TYPES[typ])
    plan = ck.KvAttention(8, 2, 128, 1, sq.tokens, chunk, 100 + chunk)
    out, lse = torch.zeros_like(q), torch.zeros(sq.tokens, 8, device=gpu)
    plan.run(cache, b, q, out=out, lse=lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.run(cache, b, q, out=out, lse=lse)
    for turn in range(4):
        _shift(sq, cache, "v", range(0, 100 + chunk // 2), -26 if turn % 2 == 0 else 26)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), lse.clone()
        _check_rows(sq, cache, q, *got, 4, 0)
        plan.run(cache, b, q, out=out, lse=lse)
        torch.cuda.synchronize()
        assert torch.equal(out, got[0]) and torch.equal(lse, got[1])
