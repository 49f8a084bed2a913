"""Heads turned in place: the stride of an axis with one entry may be anything, and differ; any
other must be the input's own."""
import pytest
import torch

import checkers_amd as ck

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,own,other", [((1, 3, 64), (192, 64, 1), (7, 64, 1)), ((5, 1, 64), (64, 64, 1), (64, 3, 1)),
                                             ((1, 5, 2, 64), (640, 128, 64, 1), (0, 128, 64, 1)), ((4, 1, 2, 64), (128, 128, 64, 1), (128, 5, 64, 1))])
def test_axes_of_one_entry(gpu, shape, own, other):
    print(f"[case] {shape} {other}", flush=True)
    rot = ck.Rotary(64)
    q = torch.randn(640, device=gpu).as_strided(shape, own)
    at = torch.arange(shape[-3], dtype=torch.int32, device=gpu) + 3
    want = ck.rotary(rot, at, q)
    back = ck.rotary(rot, at, q, out=q.as_strided(shape, other))
    torch.cuda.synchronize()
    assert torch.equal(q, want) and back.data_ptr() == q.data_ptr()


def test_others_are_refused(gpu):
    q = torch.randn(4, 4, 64, device=gpu)
    with pytest.raises(ck.CkrError, match="in place"):
        ck.rotary(ck.Rotary(64), torch.arange(4, dtype=torch.int32, device=gpu), q, out=q.transpose(0, 1))
