"""Attention of few rows over a cache in 4 bits where blocks take many items: stretches of the
line of key tiles that begin and end anywhere, also between two items' tiles, where an item
counts for more tiles than it has; up to 96 rows; more sequences than a block has threads."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests import kv4_oracle as k4
from tests import kv_oracle as ko
from tests.test_gpu_kv4 import TYPES, _attend, _batch, _bytes, _cache, _check, _fill, _i32, _values

pytestmark = pytest.mark.gpu

# a plan for one token over 32 leaves few blocks: an item's 16 tiles of padding count from 32 tiles a block on
PADDED = [
    # q type, kv heads, group, dim, page, starts, lens, window
    ("bf16", 8, 4, 128, 16, [300, 5, 700, 0, 64], [1, 1, 1, 1, 1], 0),
    ("f16", 8, 4, 64, 64, [900, 1, 31, 32, 33, 500], [1, 2, 1, 1, 3, 1], 0),
    ("bf16", 4, 4, 256, 32, [400, 1000], [1, 1], 0),
    ("bf16", 8, 2, 128, 64, [1500, 20, 700], [1, 12, 8], 0),
    ("f16", 8, 4, 128, 16, [600, 0, 0, 200], [9, 0, 1, 5], 0),
    ("bf16", 8, 1, 96, 16, [1000, 800], [3, 20], 100),
    ("bf16", 16, 8, 64, 32, [600, 90], [2, 1], 0),
    ("f16", 4, 5, 224, 16, [700, 30, 300], [4, 1, 2], 50),
]


@pytest.mark.parametrize("case", PADDED, ids=lambda c: "-".join(map(str, c[:5])))
def test_items_that_count_for_more_tiles(gpu, case):
    typ, heads, group, dim, page, starts, lens, window = case
    print(f"[case] padded {case}", flush=True)
    sq, cache, b, q, big, want, lse = _attend(gpu, *case)
    _check(sq, cache, q, want, lse, group, window)
    plan = ck.KvAttention(heads * group, heads, dim, 1, 1, 1, 32)
    dp = 64 if dim <= 64 else 128 if dim <= 128 else 256
    blocks = (plan.ws_bytes - 768 * 4) // (8 + dp * 4) // 32
    tiles = heads * sum(-(-n * group // 16) * max(1, (o + n + 31) // 32) for o, n in zip(starts, lens) if n)
    if not window:
        assert tiles >= blocks * 32, (tiles, blocks)
    first = None
    for turn in range(3):       # parts and counters left in order, whatever ran between
        out = torch.full_like(q, 9.0)
        lse = torch.full((sq.tokens, heads * group), 9.0, device=gpu)
        plan.run(cache, b, q, window=window, out=out, lse=lse)
        torch.cuda.synchronize()
        _check(sq, cache, q, out, lse, group, window)
        assert first is None or torch.equal(out, first)
        first = out
        small = ck.KvBatch(b.page_table[:1], _i32([2], gpu), _i32([0, 1], gpu), 1, 1, 3)
        plan.run(cache, small, q[:1])


@pytest.mark.parametrize("shape", [
    # q type, kv heads, group, dim, page, starts, lens, window, columns of the table
    ("bf16", 2, 4, 128, 64, [300, 5], [12, 12], 0, None),           # 48 rows
    ("f16", 1, 8, 64, 16, [700], [6], 0, None),
    ("bf16", 1, 1, 128, 16, [100, 0], [33, 47], 0, None),
    ("f16", 2, 3, 96, 32, [60, 0, 200], [15, 1, 16], 20, None),
    ("bf16", 32, 2, 64, 64, [1100, 1030, 1200, 1024], [40, 33, 25, 48], 0, None),   # 96, over a thousand keys
    ("bf16", 2, 4, 128, 64, [300, 5], [24, 17], 0, 2048),           # a hint of 131072 keys: few rows too
    ("f16", 2, 4, 128, 16, [90], [24], 0, 8192),
    ("f16", 1, 2, 64, 64, [0, 64, 500], [48, 40, 26], 0, 4096),
    ("bf16", 1, 4, 256, 16, [40], [20], 0, 8192),
], ids=lambda c: "-".join(map(str, c[:5])))
def test_up_to_96_rows(gpu, shape):
    *case, width = shape
    typ, heads, group, dim, page, starts, lens, window = case
    print(f"[case] rows {shape}", flush=True)
    if width is None:
        sq, cache, b, q, plan, out, lse = _attend(gpu, *case)
    else:
        sq = ko.Seqs(starts, lens, page, seed=3, width=width)
        cache = _cache(sq, heads, dim, gpu)
        b = _batch(sq, gpu)
        b = ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, max(lens), width * page)
        _fill(sq, cache, b, heads, dim, gpu, 3)
        q = torch.randn(sq.tokens, heads * group, dim, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(TYPES[typ])
        plan = ck.KvAttention(heads * group, heads, dim, len(starts), sq.tokens, max(lens), width * page)
        lse = torch.full((sq.tokens, heads * group), 9.0, device=gpu)
        out = plan.run(cache, b, q, lse=lse)
    torch.cuda.synchronize()
    _check(sq, cache, q, out, lse, group, window)
    ck.profile_begin()
    again = plan.run(cache, b, q, window=window)
    torch.cuda.synchronize()
    assert "kv_attention_few" in ck.profile_end() and torch.equal(again, out)


def test_more_sequences_than_threads(gpu):
    """1100 sequences, many of them empty or of one token, through kv_append, kv_read and the attention."""
    r = np.random.default_rng(5)
    n = 1100
    lens = [int(x) for x in r.choice([0, 0, 1, 1, 1, 2, 9], n)]
    starts = [int(x) for x in r.choice([0, 1, 15, 16, 40], n)]
    lens[0] = lens[-1] = 0
    lens[600:900] = [0] * 300
    heads, group, dim, page = 2, 2, 64, 16
    sq = ko.Seqs(starts, lens, page, seed=1)
    cache = _cache(sq, heads, dim, gpu)
    b = _batch(sq, gpu)
    _fill(sq, cache, b, heads, dim, gpu, 3)
    g = torch.Generator(device=gpu).manual_seed(4)
    q, k, v = (torch.randn(sq.tokens, h, dim, generator=g, device=gpu).to(torch.bfloat16) for h in (heads * group, heads, heads))
    rot = ck.Rotary(dim)
    before = [_bytes(t).clone() for t in cache.tensors()]
    turned = ck.kv_append(cache, b, rot, k, v, q=q)
    at = torch.tensor([o + i for o, x in zip(starts, lens) for i in range(x)], dtype=torch.int32, device=gpu)
    assert torch.equal(turned, ck.rotary(rot, at, q))
    # the keys as kv_write of the turned ones in 32 bits stores them, token by token
    kk = ck.rotary(rot, at, k.float())
    codes = [k4.quantise(x.cpu().float()) for x in (kk, v)]
    back = ck.kv_read(cache, b, ck.F32)
    for (c, byte), x, old, name in zip(codes, back, before, ("k", "v")):
        power = torch.exp2(byte.double() - 127)
        assert torch.equal(x.cpu().double(), (c * power.repeat_interleave(32, -1)))
    plan = ck.KvAttention(heads * group, heads, dim, n, sq.tokens, max(lens), 60)
    lse = torch.full((sq.tokens, heads * group), 9.0, device=gpu)
    out = plan.run(cache, b, turned, lse=lse)
    torch.cuda.synchronize()
    _check(sq, cache, turned, out, lse, group, 0)
    # the same tokens taken many rows at a time
    wide = ck.KvBatch(b.page_table, b.starts, b.offsets, sq.tokens, 200, 60)
    lse2 = torch.full_like(lse, 9.0)
    out = ck.KvAttention(heads * group, heads, dim, n, sq.tokens, 200, 60).run(cache, wide, turned, lse=lse2)
    torch.cuda.synchronize()
    _check(sq, cache, turned, out, lse2, group, 0)


@pytest.mark.parametrize("dim,lens", [(256, [40]), (128, [100]), (128, [20]), (64, [60])])
@pytest.mark.parametrize("first", ["unmapped", "zeros"])
def test_scores_where_the_first_keys_have_no_scale(gpu, dim, lens, first):
    """float16 queries whose first keys have no scale and whose values are too small for the output:
    the scores' log-sums are as ever."""
    print(f"[case] log-sums {dim} {lens} {first}", flush=True)
    sq = ko.Seqs([600], lens, 16, seed=2)
    cache = _cache(sq, 2, dim, gpu)
    _fill(sq, cache, _batch(sq, gpu), 2, dim, gpu, 3)
    _bytes(cache.v_scale)[:] -= 60
    for j in range(230):
        p, slot = sq.place(0, j)
        for t in (cache.k, cache.v):
            _bytes(t)[p, :, slot] = 0
        for t in (cache.k_scale, cache.v_scale):
            _bytes(t)[p, :, :, slot] = 0
    if first == "unmapped":
        sq.table[0, :14] = -1
    q = torch.randn(sq.tokens, 8, dim, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu).to(torch.float16)
    lse = torch.full((sq.tokens, 8), 9.0, device=gpu)
    out = ck.KvAttention(8, 2, dim, 1, sq.tokens, max(lens), 700).run(cache, _batch(sq, gpu), q, lse=lse)
    torch.cuda.synchronize()
    _check(sq, cache, q, out, lse, 4, 0)
    assert torch.isfinite(out).all()
