"""Forward-mode derivatives of rotary on the GPU: the tangent is what rotary makes of it."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import checkers_amd as ck

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("inverse", [False, True])
def test_rotary_turns_tangents(gpu, typ, inverse):
    rot = ck.Rotary(32, interleaved=inverse)
    g = torch.Generator(device=gpu).manual_seed(1)
    q, k, t, u = (torch.randn(2, 50, h, 40, generator=g, device=gpu).to(typ) for h in (6, 2, 6, 2))
    at = torch.arange(50, dtype=torch.int32, device=gpu) * 1000
    with fw.dual_level():
        a, b = ck.rotary(rot, at, fw.make_dual(q, t), fw.make_dual(k, u), inverse=inverse)
        got = [fw.unpack_dual(x) for x in (a, b)]
        with pytest.raises(ck.CkrError, match="tangents"):
            ck.rotary(rot, at, fw.make_dual(q, t), out=torch.empty_like(q))
        with pytest.raises(ck.CkrError, match="forward-mode"):
            ck.add_rms_norm(fw.make_dual(q[0, 0], t[0, 0]), None, torch.ones(40, dtype=typ, device=gpu))
    torch.cuda.synchronize()
    for x, want, tangent in zip(got, ck.rotary(rot, at, q, k, inverse=inverse), ck.rotary(rot, at, t, u, inverse=inverse)):
        assert torch.equal(x.primal, want) and torch.equal(x.tangent, tangent)


def test_forward_over_reverse(gpu):
    rot = ck.Rotary(16)
    x, t = (torch.randn(30, 3, 16, device=gpu) for _ in range(2))
    at = torch.arange(30, dtype=torch.int32, device=gpu)
    with fw.dual_level():
        d = fw.make_dual(x.requires_grad_(), t)
        g, = torch.autograd.grad(ck.rotary(rot, at, d).pow(3).sum(), d, create_graph=True)
        got = fw.unpack_dual(g).tangent.detach()
    with torch.no_grad():
        want = ck.rotary(rot, at, 6 * ck.rotary(rot, at, x) * ck.rotary(rot, at, t), inverse=True)
    # the same products in another order: a few roundings of 32 bits of terms of at most the largest
    assert (got - want).abs().max() <= 16 * 2.0 ** -24 * want.abs().max()
