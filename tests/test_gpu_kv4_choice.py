"""Which kernel attention over a cache in 4 bits takes chunks of 49 to 96 rows a head by: the few
rows' one reads the keys once for each 16 rows, which pays where there is much to read and
too few sequences to fill the card."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests.test_gpu_kv4 import _i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,context,rows,window,few", [
    (16, 4096, 48, 0, True), (64, 4096, 48, 0, True), (16, 4096, 96, 0, True), (16, 4096, 64, 1024, True), (1, 32768, 64, 0, True),
    (64, 4096, 96, 0, False), (64, 4096, 64, 1024, False), (16, 4096, 64, 256, False), (1, 32768, 64, 1024, False), (1, 2000, 64, 0, False),
    (64, 4096, 48, 256, True), (16, 4096, 100, 0, False)])
def test_a_window_counts_as_the_context(gpu, seqs, context, rows, window, few):
    print(f"[case] {seqs} {context} {rows} {window}", flush=True)
    heads, group, page = 8, 4, 64
    cache = ck.KvCache.empty(2, page, heads, 128, ck.F4)
    chunk = rows // group
    width = -(-(context + chunk) // page)
    b = ck.KvBatch(_i32(np.zeros((seqs, width)), gpu), _i32([context] * seqs, gpu), _i32(np.arange(seqs + 1) * chunk, gpu), seqs * chunk, chunk, context + chunk)
    q = torch.zeros(seqs * chunk, heads * group, 128, dtype=torch.bfloat16, device=gpu)
    plan = ck.KvAttention(heads * group, heads, 128, seqs, seqs * chunk, chunk, context + chunk)
    torch.cuda.synchronize()
    ck.profile_begin()
    plan.run(cache, b, q, window=window)
    torch.cuda.synchronize()
    assert ("kv_attention_few" in ck.profile_end()) == few
