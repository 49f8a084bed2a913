"""Attention with scores so large that their last bit is worth powers of two: the largest one's
value comes out, not an infinity or NaN."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu

CACHES = {"f8": ck.F8, "i8": ck.I8, "bf16": ck.BF16, "f16": ck.F16, "f4": ck.F4}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


@pytest.mark.parametrize("tokens", [1, 4, 25, 100, 300])      # 4 query heads: few, many and very many rows
@pytest.mark.parametrize("typ,cached,dim", [("bf16", "f8", 128), ("bf16", "i8", 64), ("f16", "f8", 64), ("f16", "i8", 128), ("bf16", "bf16", 128),
                                            ("f16", "f16", 64), ("bf16", "f4", 128), ("f16", "f4", 64), ("bf16", "f4", 64), ("f16", "f4", 128)])
def test_the_largest_score_wins(gpu, typ, cached, dim, tokens):
    """A key of 2^15 among keys of at most 3/4 of that, queries of 2^14 and up: scores of 2^29, in powers of
    two 32 from one float to the next, and 2^27 between the largest and the others."""
    print(f"[case] {typ} {cached} {dim} {tokens}", flush=True)
    old = 200
    sq = ko.Seqs([old], [tokens], 64, seed=1)
    n = old + tokens
    g = torch.Generator(device=gpu).manual_seed(tokens)
    k = torch.zeros(n, 1, dim, device=gpu)
    k[:, 0, 0] = 2.0 ** 14 * (torch.randint(0, 2, (n,), generator=g, device=gpu) + 0.5)     # 2^13 or 1.5 * 2^14, as 4 bits hold them
    k[7, 0, 0] = 2.0 ** 15
    v = torch.randn(n, 1, dim, generator=g, device=gpu)
    cache = ck.KvCache.empty(sq.n_pages, 64, 1, dim, CACHES[cached])
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)
    table = i32(sq.table)
    whole = ck.KvBatch(table, i32([0]), i32([0, n]), n)
    ck.kv_write(cache, whole, k, v)
    b = ck.KvBatch(table, i32(sq.starts), i32(sq.offsets), tokens, tokens, n)
    q = torch.zeros(tokens, 4, dim, device=gpu)
    q[..., 0] = 2.0 ** 14 * (1 + torch.randint(0, 128, (tokens, 4), generator=g, device=gpu) / 128)
    q = q.to(TYPES[typ])
    lse = torch.zeros(tokens, 4, device=gpu)
    out = ck.KvAttention(4, 1, dim, 1, tokens, tokens, n).run(cache, b, q, scale=1.0, lse=lse)
    back = ck.kv_read(cache, whole, ck.F32)[1][7, 0]
    torch.cuda.synchronize()
    # of one weight and 32-bit sums: the weight's rounding (8 bits over bfloat16, 11 elsewhere) and the output's
    unit = 1.01 * (ko.UNIT[q.dtype] + (2.0 ** -8 if cached == "bf16" else 2.0 ** -11))
    assert ((out.float() - back).abs() <= unit * back.abs() + 2.0 ** -24).all()
    want = q[..., 0].double() * ck.kv_read(cache, whole, ck.F32)[0][7, 0, 0].double()
    # a float's product and its scale by log2 e, and what a last bit of 2^29.5 is against the maximum
    assert ((lse.double() - want).abs() <= 2.0 ** -21 * want).all()
