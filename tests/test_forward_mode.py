"""Forward-mode derivatives: rotary turns tangents, the operators without a derivative
refuse them (on the CPU, with the call of the kernel replaced by the formula)."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import checkers_amd as ck
from checkers_amd import kv


class _Plain:
    """What a Rotary is to rotary(): one turn of pi / 2 a position, halves apart."""
    pairs = 2


def _turn(rotary, positions, xs, outs, inverse, stream):
    for x, y in zip(xs, outs):
        assert x.stride(-1) == 1 and not fw.unpack_dual(x).tangent is not None
        half = rotary.pairs
        c = torch.tensor([1.0, 0, -1, 0])[positions.long() % 4][:, None, None]
        s = torch.tensor([0.0, 1, 0, -1])[positions.long() % 4][:, None, None] * (-1 if inverse else 1)
        a, b = x[..., :half], x[..., half:2 * half]
        with torch.no_grad():
            y.copy_(torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * half:]), -1))


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(kv, "_rotate", _turn)
    return _Plain(), torch.tensor([0, 1, 2, 3, 5], dtype=torch.int32)


def _of(rot, at, x, inverse=False):
    y = torch.empty_like(x)
    _turn(rot, at, (x,), (y,), inverse, None)
    return y


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("no_grad", [False, True])
def test_rotary_turns_tangents(plain, inverse, no_grad):
    rot, at = plain
    q, k, t, u = (torch.randn(5, h, 6) for h in (3, 2, 3, 2))
    with fw.dual_level(), torch.set_grad_enabled(not no_grad):
        a, b = ck.rotary(rot, at, fw.make_dual(q, t), fw.make_dual(k, u), inverse=inverse)
        assert torch.equal(fw.unpack_dual(a).tangent, _of(rot, at, t, inverse)) and torch.equal(fw.unpack_dual(b).tangent, _of(rot, at, u, inverse))
        assert torch.equal(fw.unpack_dual(a).primal, _of(rot, at, q, inverse))
        # of one input only, and of a tangent laid out another way
        a, b = ck.rotary(rot, at, q, fw.make_dual(k, u.transpose(1, 2).contiguous().transpose(1, 2)), inverse=inverse)
        assert torch.equal(fw.unpack_dual(b).tangent, _of(rot, at, u, inverse))
        tangent = fw.unpack_dual(a).tangent
        assert tangent is None or not tangent.any()
        one = ck.rotary(rot, at, fw.make_dual(q, t))
        assert torch.equal(fw.unpack_dual(one).tangent, _of(rot, at, t))


def test_forward_over_reverse(plain):
    """A Hessian times a vector of sum(rotary(x)^3)."""
    rot, at = plain
    x, t = torch.randn(5, 2, 4), torch.randn(5, 2, 4)
    with fw.dual_level():
        d = fw.make_dual(x.requires_grad_(), t)
        g, = torch.autograd.grad(ck.rotary(rot, at, d).pow(3).sum(), d, create_graph=True)
        got = fw.unpack_dual(g).tangent
    want = _of(rot, at, 6 * _of(rot, at, x.detach()) * _of(rot, at, t), inverse=True)
    assert torch.allclose(got, want)


def test_outside_of_a_level_nothing_changes(plain):
    rot, at = plain
    x = torch.randn(5, 2, 4)
    assert torch.equal(ck.rotary(rot, at, x), _of(rot, at, x))


def test_refusals(plain):
    rot, at = plain
    x = torch.randn(5, 2, 6)
    with fw.dual_level(), torch.no_grad():
        d = fw.make_dual(x, x)

        class Sizes:
            n_tokens, n_heads, head_dim = 5, 2, 6

        plan = object.__new__(ck.KvAttention)
        calls = (lambda: ck.rotary(rot, at, d, out=x), lambda: ck.kv_write(Sizes, Sizes, d, x), lambda: ck.kv_write(Sizes, Sizes, x, d),
                 lambda: ck.kv_append(Sizes, Sizes, None, x, x, q=d), lambda: plan.run(Sizes, Sizes, d),
                 lambda: ck.add_rms_norm(d[0], None, x[0, 0]), lambda: ck.add_rms_norm(x[0], d[0], x[0, 0]), lambda: ck.add_rms_norm(x[0], None, d[0, 0]))
        for call in calls:
            with pytest.raises(ck.CkrError, match="tangent|forward-mode"):
                call()


@pytest.mark.parametrize("order", [(0, 1, 2), (1, 0, 2)])
def test_one_layout_with_and_without_gradients(plain, order):
    """Heads that lie before tokens: the output is contiguous whether a gradient is recorded, a
    tangent turned, or neither."""
    rot, at = plain
    x = torch.randn(*(torch.empty(5, 3, 6).permute(order).shape)).permute(order)
    with torch.no_grad():
        want = ck.rotary(rot, at, x)
    with fw.dual_level():
        dual = fw.unpack_dual(ck.rotary(rot, at, fw.make_dual(x, torch.randn(5, 3, 6)))).primal
    for y in (want, dual, ck.rotary(rot, at, x.detach().requires_grad_())):
        assert y.is_contiguous() and y.stride() == want.stride() and torch.equal(y, want)
