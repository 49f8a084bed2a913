"""Calls of so many tokens that a block takes several one after another (rotary from 2048 tokens of
40 heads on, kv_append and kv_read alike): bit for bit what small calls make of the same tokens,
in which a block takes its tokens side by side only."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests.test_gpu_kv4 import _bytes, _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,tokens,heads,dim,rotary_dim,interleaved", [
    (torch.bfloat16, 9001, (32, 8), 128, 128, False), (torch.bfloat16, 9001, (32, 8), 128, 128, True), (torch.float16, 4099, (36, 4), 96, 40, False),
    (torch.float32, 8197, (20, 4), 80, 20, False), (torch.float32, 6145, (20, 4), 80, 20, True), (torch.bfloat16, 33001, (4, 2), 72, 36, False),
    (torch.float32, 4097, (3, 3), 1024, 1024, False)])
def test_rotary(gpu, typ, tokens, heads, dim, rotary_dim, interleaved):
    print(f"[case] rotary {typ} {tokens} {heads} {dim} {rotary_dim} {interleaved}", flush=True)
    rot = ck.Rotary(rotary_dim, interleaved=interleaved)
    g = torch.Generator(device=gpu).manual_seed(tokens)
    q, k = (torch.randn(tokens, h, dim, generator=g, device=gpu).to(typ) for h in heads)
    at = torch.randint(0, 1 << 20, (tokens,), generator=g, device=gpu).to(torch.int32)
    piece = 300
    want = [torch.cat(x) for x in zip(*(ck.rotary(rot, at[i:i + piece], q[i:i + piece], k[i:i + piece]) for i in range(0, tokens, piece)))]
    got = ck.rotary(rot, at, q, k)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ck.rotary(rot, at, q, k, out=(q, k))         # in place, loads of several tokens ahead of stores
    torch.cuda.synchronize()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def _pieces(table, starts, lens, most, gpu):
    """The batch in calls of at most `most` tokens: (rows of the packed tensors, batch)."""
    at = 0
    for s, (o, n) in enumerate(zip(starts, lens)):
        for i in range(0, n, most):
            m = min(most, n - i)
            yield slice(at + i, at + i + m), ck.KvBatch(table[s:s + 1], _i32([o + i], gpu), _i32([0, m], gpu), m)
        at += n


@pytest.mark.parametrize("cached,typ,dim,rotary_dim,interleaved,heads", [
    (ck.F4, torch.bfloat16, 128, 128, False, (32, 8)), (ck.F4, torch.float32, 96, 32, False, (8, 2)), (ck.F4, torch.float16, 64, 64, True, (16, 4)),
    (ck.F8, torch.bfloat16, 128, 64, False, (32, 8)), (ck.I8, torch.float32, 80, 40, False, (8, 2)), (ck.BF16, torch.bfloat16, 128, 128, True, (16, 4))])
def test_append_and_read(gpu, cached, typ, dim, rotary_dim, interleaved, heads):
    print(f"[case] append {cached} {typ} {dim} {rotary_dim} {interleaved}", flush=True)
    page, lens = 64, [9000, 0, 1, 70, 30011, 0, 3999, 17]
    starts = [5, 0, 63, 1000, 0, 7, 64, 30]
    n, width = sum(lens), max(-(-(o + x) // page) for o, x in zip(starts, lens))
    r = np.random.default_rng(1)
    need = [-(-(o + x) // page) for o, x in zip(starts, lens)]
    ids, table, used = r.permutation(sum(need)), np.full((len(lens), width), -1, np.int32), 0
    for s, p in enumerate(need):
        table[s, :p] = ids[used:used + p]
        used += p
    table[0, 20] = -1                                        # not mapped: not stored, reads as zeros
    table[4, 100] = sum(need) + 5
    table = _i32(table, gpu)
    g = torch.Generator(device=gpu).manual_seed(2)
    q, k, v = (torch.randn(n, h, dim, generator=g, device=gpu).to(typ) for h in (heads[0], heads[1], heads[1]))
    rot = ck.Rotary(rotary_dim, interleaved=interleaved)
    one, many = (ck.KvCache.empty(sum(need), page, heads[1], dim, cached) for _ in range(2))
    batch = ck.KvBatch(table, _i32(starts, gpu), _i32(np.concatenate([[0], np.cumsum(lens)]), gpu), n)
    want = torch.empty_like(q)
    for rows, b in _pieces(table, starts, lens, 500, gpu):
        ck.kv_append(many, b, rot, k[rows], v[rows], q=q[rows], out=want[rows])
    ck.kv_append(one, batch, rot, k, v, q=q, out=q)          # in place
    torch.cuda.synchronize()
    assert torch.equal(q, want)
    for a, b in zip(one.tensors(), many.tensors()):
        assert torch.equal(_bytes(a) if a.element_size() == 1 else a, _bytes(b) if b.element_size() == 1 else b)
    tag = {torch.bfloat16: ck.BF16, torch.float16: ck.F16, torch.float32: ck.F32}[typ]
    got = ck.kv_read(one, batch, tag)
    for rows, b in _pieces(table, starts, lens, 500, gpu):
        for x, y in zip(got, ck.kv_read(many, b, tag)):
            assert torch.equal(x[rows], y)
