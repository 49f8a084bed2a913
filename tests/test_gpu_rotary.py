"""Rotary positions: rotary and its gradients against formulas in 64 bits and differences,
kv_append against the two operators that it joins."""
import math

import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests import kv4_oracle as k4
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SCALINGS = {"none": None, "linear": dict(kind="linear", factor=4.0), "base": dict(kind="base", factor=2.0),
            "bands": dict(kind="bands", factor=8.0, length=8192), "yarn": dict(kind="yarn", factor=16.0, length=4096)}


def _i32(a, gpu):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=gpu)


def _expected(scaling, rot, base):
    if scaling == "linear":
        return [f / 4 for f in k4.frequencies(rot, base)], 1.0
    if scaling == "base":
        return k4.frequencies(rot, base * 2 ** (rot / (rot - 2))), 1.0
    if scaling == "bands":
        return k4.bands(rot, base, 8.0, 8192), 1.0
    if scaling == "yarn":
        return k4.yarn(rot, base, 16.0, 4096)
    return k4.frequencies(rot, base), 1.0


def _bound(y, size, typ):
    """Cosine and sine are rounded once (and their angles are off by 2^-30 at most), products and
    their sum too: 4 roundings of 32 bits of the terms' size, then one to the type."""
    return 4.5 * ko.U32 * size + ko.UNIT[TYPES[typ]] * 1.01 * y.abs() + 2.0 ** -25


@pytest.mark.parametrize("scaling", list(SCALINGS))
@pytest.mark.parametrize("rot,base", [(128, 500000.0), (64, 10000.0), (20, 10000.0)])
def test_frequencies_of_scalings(gpu, scaling, rot, base):
    r = ck.Rotary(rot, base, scaling=SCALINGS[scaling])
    f, m = _expected(scaling, rot, base)
    assert r.rotary_dim == rot and r.magnitude == pytest.approx(m, rel=1e-15)
    assert np.allclose(r.frequencies, f, rtol=1e-12, atol=0)
    turns = r.turns.cpu().numpy().view(np.uint64).astype(np.float64) * 2.0 ** -64
    # a turn is kept to 2^-64, so off by 2^-65 at most (1.1e-12 of the smallest here, 2.4e-8), besides 1e-12 as above
    assert np.allclose(turns, np.array(f) / (2 * math.pi), rtol=1e-12, atol=2.0 ** -65)


CASES = [
    # type, lead (batch, tokens), q heads, k heads, dim, rot, interleaved, order, far
    ("bf16", (64,), 32, 8, 128, 128, False, "thd", 120000),
    ("bf16", (1,), 4, 0, 128, 128, True, "thd", 5),
    ("f16", (3, 37), 8, 2, 96, 96, False, "bthd", 0),
    ("f32", (2, 50), 3, 3, 80, 20, True, "bhtd", 1000),
    ("f32", (7,), 5, 1, 80, 20, False, "thd", 1 << 30),
    ("bf16", (2, 9), 6, 2, 40, 36, False, "bhtd", 2000000),
    ("f16", (11,), 2, 1, 33, 6, True, "thd", 100),
    ("f32", (13,), 1, 1, 2, 2, False, "thd", 100),
    ("bf16", (5,), 7, 3, 250, 250, True, "thd", 70000),
    ("bf16", (6,), 2, 2, 1024, 1000, False, "thd", 9),
    ("f16", (300,), 40, 40, 64, 64, False, "thd", 0),
    ("bf16", (2000,), 1, 0, 128, 64, False, "thd", 0),
    ("f32", (4, 1), 2, 1, 256, 2, False, "bthd", 50000),
]


def _inputs(gpu, typ, lead, heads, dim, order, seed):
    g = torch.Generator(device=gpu).manual_seed(seed)
    shape = (*lead, heads, dim)
    if order == "bhtd":
        return torch.randn(lead[0], heads, lead[1], dim, generator=g, device=gpu).to(TYPES[typ]).transpose(1, 2)
    return torch.randn(shape, generator=g, device=gpu).to(TYPES[typ])


def _positions(gpu, lead, far):
    r = np.random.default_rng(3)
    return _i32(r.integers(0, far, lead) if far else np.broadcast_to(np.arange(lead[-1]), lead).copy(), gpu)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("scaling", ["none", "yarn"])
def test_rotary(gpu, case, scaling):
    print(f"[case] rotary {case} {scaling}", flush=True)
    typ, lead, hq, hk, dim, rot, inter, order, far = case
    if scaling == "yarn" and rot <= 2:
        pytest.skip("one pair")
    r = ck.Rotary(rot, 10000.0, interleaved=inter, scaling=SCALINGS[scaling])
    pos = _positions(gpu, lead, far)
    xs = [_inputs(gpu, typ, lead, h, dim, order, 10 + h) for h in (hq, hk) if h]
    for inverse in (False, True):
        got = ck.rotary(r, pos, *xs, inverse=inverse)
        got = got if len(xs) == 2 else (got,)
        torch.cuda.synchronize()
        for x, y in zip(xs, got):
            assert y.dtype == x.dtype and y.shape == x.shape
            want, size = k4.turned(x.cpu(), pos.cpu(), rot, inter, r.frequencies, r.magnitude, inverse)
            assert ((y.cpu().double() - want).abs() <= _bound(want, size, typ)).all()
            assert torch.equal(y[..., rot:], x[..., rot:])
    # in place, and into slices of a wider tensor
    copies = [x.clone() for x in xs]
    again = ck.rotary(r, pos, *copies, out=copies[0] if len(xs) == 1 else tuple(copies), inverse=True)
    again = again if len(xs) == 2 else (again,)
    wide = torch.full((*lead, hq + hk + 1, dim + 3), 7.0, dtype=TYPES[typ], device=gpu)
    parts = [wide[..., 1:1 + hq, 1:1 + dim], wide[..., 1 + hq:, 1:1 + dim]][:len(xs)]
    ck.rotary(r, pos, *xs, out=parts[0] if len(xs) == 1 else tuple(parts), inverse=True)
    torch.cuda.synchronize()
    for y, z, p, c in zip(got, again, parts, copies):
        assert z is c and torch.equal(y, z) and torch.equal(y, p)
    assert (wide[..., 0, :] == 7).all() and (wide[..., 0] == 7).all() and (wide[..., 1 + dim:] == 7).all()


def test_rotary_positions_shared_by_the_batch_and_negative_ones(gpu):
    r = ck.Rotary(64)
    q = torch.randn(3, 5, 2, 64, device=gpu)
    pos = _i32([0, -1, 2**31 - 1, -2**31, 7], gpu)
    got = ck.rotary(r, pos, q)
    each = ck.rotary(r, pos[None].expand(3, 5), q)
    assert torch.equal(got, each)
    f = [math.fmod(x, 2 * math.pi) for x in r.frequencies]
    for t, p in enumerate([0, -1, 2**31 - 1, -2**31, 7]):   # the angle by whole numbers: turns of 2^-64
        turns = [int(v) for v in r.turns.cpu().numpy().view(np.uint64)]
        a = torch.tensor([(p * n) % 2**64 / 2**64 * 2 * math.pi for n in turns], dtype=torch.float64)
        x = q[:, t].cpu().double()
        want = torch.cat((x[..., :32] * a.cos() - x[..., 32:] * a.sin(), x[..., 32:] * a.cos() + x[..., :32] * a.sin()), -1)
        assert ((got[:, t].cpu().double() - want).abs() <= 5 * ko.U32 * (x.abs() + x.roll(32, -1).abs())).all(), p
    assert len(f) == 32


@pytest.mark.parametrize("typ,lead,dim,rot,inter", [("f32", (6,), 20, 12, False), ("f32", (2, 5), 16, 16, True), ("bf16", (2, 33), 64, 48, False),
                                                    ("f16", (40,), 128, 128, True)])
def test_gradients(gpu, typ, lead, dim, rot, inter):
    r = ck.Rotary(rot, 100.0, interleaved=inter, scaling=dict(kind="yarn", factor=4.0, length=64))
    pos = _positions(gpu, lead, 500)
    q, k = (_inputs(gpu, typ, lead, h, dim, "thd", h).requires_grad_() for h in (3, 2))
    gq, gk = (_inputs(gpu, typ, lead, h, dim, "thd", 20 + h) for h in (3, 2))
    y = ck.rotary(r, pos, q, k)
    got = torch.autograd.grad(y, (q, k), (gq, gk))
    for g, d in zip((gq, gk), got):     # the formula's: the transposed matrix
        want, size = k4.turned(g.cpu(), pos.cpu(), rot, inter, r.frequencies, r.magnitude, True)
        assert ((d.cpu().double() - want).abs() <= _bound(want, size, typ)).all()
    if typ == "f32":                     # differences: the operator is linear, so a whole step is exact but for roundings
        step = torch.randn_like(q)
        with torch.no_grad():
            diff = ck.rotary(r, pos, q + step) - ck.rotary(r, pos, q - step)
        a, b = (diff.double() * gq.double()).sum(), 2 * (step.double() * got[0].double()).sum()
        n = q.numel()
        assert abs(a - b) <= 16 * ko.U32 * 2 * r.magnitude * math.sqrt(n) * 4 * math.sqrt(n)   # n products of values of a few units
    # one output used, and gradients that are expanded or lie in another order
    one, = torch.autograd.grad(ck.rotary(r, pos, q, k)[1].sum(), k)
    want, size = k4.turned(torch.ones(k.shape), pos.cpu(), rot, inter, r.frequencies, r.magnitude, True)
    assert ((one.cpu().double() - want).abs() <= _bound(want, size, typ)).all()
    turned, = torch.autograd.grad(ck.rotary(r, pos, q), q, gq.transpose(-1, -2).contiguous().transpose(-1, -2))
    assert torch.equal(turned, got[0])
    # the gradient of the gradient turns forward again
    q2 = gq.detach().requires_grad_()
    d, = torch.autograd.grad(ck.rotary(r, pos, q), q, q2, create_graph=True)
    dd, = torch.autograd.grad(d, q2, q.detach())
    with torch.no_grad():
        assert torch.equal(dd, ck.rotary(r, pos, q))
    # leaves' gradients add up over two uses
    (ck.rotary(r, pos, k).sum() + ck.rotary(r, pos, k).sum()).backward()
    assert torch.allclose(k.grad.float(), 2 * one.float(), rtol=2 * ko.UNIT[TYPES[typ]] * 2, atol=1e-6)


def test_gradients_need_positions_as_they_were(gpu):
    r, pos = ck.Rotary(32), _i32([1, 2], gpu)
    q = torch.randn(2, 1, 32, device=gpu, requires_grad=True)
    y = ck.rotary(r, pos, q).sum()
    pos += 1
    with pytest.raises(RuntimeError):
        y.backward()


def test_infinities_stay_in_their_pair(gpu):
    for inter in (False, True):
        x = torch.ones(1, 1, 64, device=gpu)
        x[0, 0, 40], x[0, 0, 5] = float("inf"), float("nan")
        y = ck.rotary(ck.Rotary(48, interleaved=inter), _i32([3], gpu), x)
        wild = (~torch.isfinite(y)).nonzero()[:, 2].tolist()
        assert wild == ([4, 5, 40, 41] if inter else [5, 16, 29, 40])


APPEND = [
    # type, cache, q heads, kv heads, dim, rot, interleaved, page, starts, lens
    ("bf16", "f8", 32, 8, 128, 128, False, 64, [1000], [1]),
    ("bf16", "f4", 8, 2, 128, 128, False, 16, [5, 0, 130, 17, 0], [1, 33, 0, 100, 257]),
    ("f16", "i8", 6, 3, 80, 32, True, 32, [5, 0, 700], [1, 50, 3]),
    ("bf16", "bf16", 4, 4, 96, 96, False, 128, [9, 70000], [40, 2]),
    ("f16", "f16", 0, 1, 64, 64, True, 16, [0, 3], [100, 1]),
    ("f32", "f4", 5, 5, 256, 256, True, 32, [100], [70]),
    ("f32", "f8", 1, 1, 16, 6, False, 16, [0], [300]),
    ("bf16", "f4", 7, 1, 32, 20, False, 16, [50, 1], [9, 1]),
    ("f16", "f4", 16, 2, 224, 72, False, 64, [0], [129]),
    ("bf16", "i8", 20, 1, 128, 2, False, 256, [3000], [65]),
    ("bf16", "f4", 64, 8, 64, 64, False, 64, [1], [400]),
    ("f16", "f8", 200, 2, 128, 64, True, 16, [8], [3]),
]
TAGS = {"f4": ck.F4, "f8": ck.F8, "i8": ck.I8, "bf16": ck.BF16, "f16": ck.F16}


def _raw(cache):
    return [t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()]).clone() for t in cache.tensors()]


@pytest.mark.parametrize("case", APPEND, ids=lambda c: "-".join(map(str, c[:8])))
def test_append_is_rotary_and_write(gpu, case):
    """The cache holds, bit for bit, what kv_write makes of the keys turned in 32 bits, and the
    queries are rotary's."""
    print(f"[case] append {case}", flush=True)
    typ, fmt, hq, hk, dim, rot, inter, page, starts, lens = case
    sq = ko.Seqs(starts, lens, page, seed=dim)
    if len(lens) > 3:
        sq.table[3, 1] = -1                    # an unmapped page
        sq.table[4, 0] = sq.n_pages + 3
    b = ck.KvBatch(_i32(sq.table, gpu), _i32(sq.starts, gpu), _i32(sq.offsets, gpu), sq.tokens)
    caches = [ck.KvCache.empty(sq.n_pages, page, hk, dim, TAGS[fmt]) for _ in range(3)]
    for c in caches:
        for t in c.tensors():
            t.view(torch.uint8).fill_(0x5a)
    r = ck.Rotary(rot, 10000.0, interleaved=inter, scaling=SCALINGS["yarn"] if rot > 2 else None)
    g = torch.Generator(device=gpu).manual_seed(7)
    qkv = torch.randn(sq.tokens, hq + 2 * hk, dim, generator=g, device=gpu).to(TYPES[typ])
    if fmt in ("f4", "f8", "i8"):
        qkv[0, hq, 1], qkv[0, hq + hk, dim - 1] = float("nan"), float("inf")
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    kept = qkv.clone()
    pos = _i32(np.concatenate([np.arange(o, o + n) for o, n in zip(starts, lens)]), gpu)
    out = ck.kv_append(caches[0], b, r, k, v, q=q if hq else None)
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(qkv), torch.nan_to_num(kept))
    ck.kv_write(caches[1], b, ck.rotary(r, pos, k.float()), v.float())
    for a, c in zip(_raw(caches[0]), _raw(caches[1])):
        assert torch.equal(a, c)
    if hq:
        assert torch.equal(out, ck.rotary(r, pos, q))
        # in place, at positions of its own
        other = _i32(np.arange(sq.tokens)[::-1].copy(), gpu)
        want = ck.rotary(r, other, q)
        got = ck.kv_append(caches[2], b, r, k, v, q=q, out=q, positions=other)
        assert got is q and torch.equal(q, want) and torch.equal(torch.nan_to_num(qkv[:, hq:]), torch.nan_to_num(kept[:, hq:]))
        ck.kv_write(caches[1], b, ck.rotary(r, other, k.float()), v.float())
    else:
        assert out is None
        ck.kv_append(caches[2], b, r, k, v)
    for a, c in zip(_raw(caches[2]), _raw(caches[1])):
        assert torch.equal(a, c)
    # nothing turned
    ck.kv_append(caches[0], b, None, k, v)
    ck.kv_write(caches[1], b, k, v)
    for a, c in zip(_raw(caches[0]), _raw(caches[1])):
        assert torch.equal(a, c)


def test_append_leaves_tokens_of_no_sequence(gpu):
    """Rows behind the last sequence (a padded batch) stay, in the output and the cache."""
    cache = ck.KvCache.empty(4, 16, 1, 64, ck.F4)
    table, starts, offsets = _i32([[0, 1], [2, 3]], gpu), _i32([3, 0], gpu), _i32([0, 2, 5], gpu)
    b = ck.KvBatch(table, starts, offsets, 9)
    q, kv = torch.randn(9, 3, 64, device=gpu), torch.randn(9, 1, 64, device=gpu)
    out = torch.full((9, 3, 64), 5.0, device=gpu)
    ck.kv_append(cache, b, ck.Rotary(64), kv, kv, q=q, out=out)
    assert (out[5:] == 5).all() and torch.equal(out[:5], ck.rotary(ck.Rotary(64), _i32([3, 4, 0, 1, 2], gpu), q[:5]))
    held = (cache.k_scale.view(torch.uint8) != 0).sum().item()
    assert held == 5 * 2


def test_a_layer_as_it_is_used_on_a_stream_and_in_a_graph(gpu):
    """Norm, append and attention of a step over a 4-bit cache, eager, on another stream and captured;
    positions move on between the replays."""
    heads, kv, dim, hidden, S = 8, 2, 64, 256, 3
    g = torch.Generator(device=gpu).manual_seed(1)
    w = (torch.randn(hidden, (heads + 2 * kv) * dim, generator=g, device=gpu) / 16).to(torch.bfloat16)
    x, one = torch.randn(S, hidden, generator=g, device=gpu).to(torch.bfloat16), torch.ones(hidden, dtype=torch.bfloat16, device=gpu)
    r = ck.Rotary(dim)
    table = torch.randperm(S * 8, generator=g, device=gpu).to(torch.int32).view(S, 8)
    starts = _i32([5, 90, 17], gpu)
    b = ck.KvBatch(table, starts, _i32([0, 1, 2, 3], gpu), S, 1, 128)
    prompts = [torch.randn(S * 100, kv, dim, generator=g, device=gpu).to(torch.bfloat16) for _ in range(2)]

    def fresh():
        c = ck.KvCache.empty(S * 8, 16, kv, dim, ck.F4)
        ck.kv_append(c, ck.KvBatch(table, _i32([0] * S, gpu), _i32([0, 100, 200, 300], gpu), 300), r, *prompts)
        return c

    cache, plan = fresh(), ck.KvAttention(heads, kv, dim, S, S, 1, 128)
    out, q_out = torch.empty(S, heads, dim, dtype=torch.bfloat16, device=gpu), torch.empty(S, heads, dim, dtype=torch.bfloat16, device=gpu)

    def step(stream=None):
        y, _, _ = ck.add_rms_norm(x, None, one, stream=stream)
        if stream is None:
            qkv = (y @ w).view(S, -1, dim)
        else:
            with torch.cuda.stream(stream):
                qkv = (y @ w).view(S, -1, dim)
        ck.kv_append(cache, b, r, qkv[:, heads:heads + kv], qkv[:, heads + kv:], q=qkv[:, :heads], out=q_out, stream=stream)
        plan.run(cache, b, q_out, out=out, stream=stream)

    step()
    torch.cuda.synchronize()
    want = out.clone()
    k, v = ck.kv_read(cache, ck.KvBatch(table, _i32([0] * S, gpu), _i32([0, 6, 97, 115], gpu), 115), ck.BF16)
    for s, (lo, hi) in enumerate(((0, 6), (6, 97), (97, 115))):   # the plain layer over what the cache holds
        kk, vv = (t[lo:hi].float().repeat_interleave(heads // kv, 1) for t in (k, v))
        p = torch.softmax((q_out[s].float()[None] * kk).sum(-1) * dim ** -0.5, 0)
        assert ((p[..., None] * vv).sum(0) - out[s].float()).abs().max() < 2 ** -8 * vv.abs().max()
    side = torch.cuda.Stream()
    out.zero_()
    torch.cuda.synchronize()
    step(side)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        starts.copy_(torch.tensor([5 + i, 90 - i, 17], dtype=torch.int32))
        x.copy_(torch.randn(S, hidden, device=gpu))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, held = out.clone(), _raw(cache)
        step()
        torch.cuda.synchronize()
        assert torch.equal(out, got) and all(torch.equal(a, c) for a, c in zip(held, _raw(cache))), i


def test_training_step_in_a_graph(gpu):
    """Forward and backward captured; every replay equals the eager gradients."""
    r, pos = ck.Rotary(64), _i32(np.arange(50), gpu)
    q, k = (torch.randn(50, h, 64, device=gpu, requires_grad=True) for h in (4, 2))
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def step():
        return torch.autograd.grad(ck.rotary(r, pos, q, k), (q, k), (gq, gk))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dq, dk = step()
    for i in range(3):
        gq.copy_(torch.randn_like(gq))
        pos.add_(i)
        graph.replay()
        torch.cuda.synchronize()
        got = dq.clone(), dk.clone()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want)), i


def test_rotary_dropped_while_another_stream_uses_it(gpu):
    """The table outlives the work that was queued on other streams."""
    side = torch.cuda.Stream()
    x, pos = torch.randn(4000, 32, 128, device=gpu), _i32(np.arange(4000), gpu)
    want = ck.rotary(ck.Rotary(128), pos, x)
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=gpu)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):
            busy = busy @ busy * 1e-3
    r = ck.Rotary(128)
    got = ck.rotary(r, pos, x, stream=side)
    del r
    torch.empty(64, dtype=torch.int64, device=gpu).fill_(0)   # what might take the table's memory
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_empty_calls(gpu):
    r = ck.Rotary(64)
    none = torch.zeros(0, 3, 64, device=gpu)
    assert ck.rotary(r, _i32([], gpu), none).shape == (0, 3, 64)
    no_heads = torch.zeros(5, 0, 64, device=gpu)
    a, b = ck.rotary(r, _i32(range(5), gpu), no_heads, no_heads)
    assert a.shape == b.shape == (5, 0, 64)
    q = torch.zeros(0, 3, 64, device=gpu, requires_grad=True)
    ck.rotary(r, _i32([], gpu), q).sum().backward()
    assert q.grad.shape == q.shape
    cache = ck.KvCache.empty(2, 16, 1, 64, ck.F4)
    batch = ck.KvBatch(_i32([[0]], gpu), _i32([0], gpu), _i32([0, 0], gpu), 0)
    assert ck.kv_append(cache, batch, r, none[:, :1], none[:, :1], q=none).shape == (0, 3, 64)


def test_refusals(gpu):
    def bad(part, f, *a, **kw):
        with pytest.raises(ck.CkrError) as e:
            f(*a, **kw)
        assert e.value.code == ck.CKR_E_INVALID and part in str(e.value), str(e.value)

    for args, part in (((7,), "even"), ((0,), "even"), ((64, -1.0), "base"), ((64, 1e4, False, dict(kind="far", factor=2)), "scaling kind"),
                       ((64, 1e4, False, dict(kind="linear")), "factor"), ((64, 1e4, False, dict(kind="linear", factor=2, length=4)), "takes"),
                       ((64, 1e4, False, dict(kind="bands", factor=2)), "length"), ((64, 1e4, False, dict(kind="bands", factor=2, length=9, low=4)), "above low"),
                       ((64, 1e4, False, dict(kind="yarn", factor=2, length=9, fast=1)), "fast"), ((2, 1e4, False, dict(kind="base", factor=2)), "two pairs")):
        bad(part, ck.Rotary, *args)
    bad("not finite", ck.Rotary.of, [1.0, float("inf")])
    bad("one pair", ck.Rotary.of, [])
    bad("magnitude", ck.Rotary.of, [1.0], magnitude=float("nan"))
    bad("GPU", ck.Rotary, 64, device="cpu")
    r, pos = ck.Rotary(64), _i32([0, 1], gpu)
    q = torch.zeros(2, 3, 64, device=gpu)
    bad("[tokens, heads, dim]", ck.rotary, r, pos, q[0])
    bad("[tokens, heads, dim]", ck.rotary, r, pos, q, q[None])
    bad("positions", ck.rotary, r, pos[:1], q)
    bad("positions", ck.rotary, r, pos.long(), q)
    bad("positions", ck.rotary, r, pos.cpu(), q)
    bad("k must be", ck.rotary, r, pos, q, q.half())
    bad("k must be", ck.rotary, r, pos, q, q[..., :32])
    bad("GPU", ck.rotary, r, pos, q.cpu())
    bad("contiguous", ck.rotary, r, pos, q.transpose(1, 2).contiguous().transpose(1, 2))
    bad("half the head size", ck.rotary, r, pos, q[..., :62])
    bad("not dtype", ck.rotary, r, pos, q.to(torch.int8))
    bad("not a type", ck.rotary, r, pos, q.double())
    bad("out of q", ck.rotary, r, pos, q, out=q[:, :2])
    bad("as many", ck.rotary, r, pos, q, q, out=(q,))
    bad("in place", ck.rotary, r, pos[:1], q[:1], out=torch.as_strided(q, (1, 3, 64), (192, 128, 1)))
    bad("overlap", ck.rotary, r, pos, q, out=q[:, :1].expand(2, 3, 64).clone()[:1].expand(2, 3, 64))
    grad = q.clone().requires_grad_()
    bad("neither", ck.rotary, r, pos, grad, out=q)
    bad("neither", ck.rotary, r, pos, grad, stream=torch.cuda.current_stream())
    bad("no gradients", ck.rotary, r, pos, q, out=grad)
    cache = ck.KvCache.empty(2, 16, 1, 64, ck.F4)
    b = ck.KvBatch(_i32([[0]], gpu), _i32([0], gpu), _i32([0, 2], gpu), 2)
    kv = torch.zeros(2, 1, 64, device=gpu)
    bad("no backward", ck.kv_append, cache, b, r, kv, kv, q=grad)
    bad("one type", ck.kv_append, cache, b, r, kv, kv.half())
    bad("q must be of k's type", ck.kv_append, cache, b, r, kv, kv, q=q.half())
    bad("out belongs", ck.kv_append, cache, b, r, kv, kv, out=q)
    bad("q must be [2", ck.kv_append, cache, b, r, kv, kv, q=q[0])
    bad("positions", ck.kv_append, cache, b, r, kv, kv, positions=pos.long())
    bad("half the head size", ck.kv_append, cache, b, ck.Rotary(66), kv, kv)
    bad("overlap", ck.kv_append, cache, b, r, kv, kv, q=q, out=q[:, :1].expand(2, 3, 64))
    bad("16-byte", ck.kv_append, cache, b, r, torch.zeros(2 * 64 + 1, device=gpu)[1:].view(2, 1, 64), kv)
    torch.cuda.synchronize()


def test_outputs_that_other_rows_are_read_from(gpu):
    """Two tensors swapped by their outputs, or written to one, would be read while they are written."""
    r, pos = ck.Rotary(64), _i32([0, 1], gpu)
    q, k, o = (torch.zeros(2, 3, 64, device=gpu) for _ in range(3))
    cache = ck.KvCache.empty(2, 16, 3, 64, ck.F4)
    b = ck.KvBatch(_i32([[0]], gpu), _i32([0], gpu), _i32([0, 2], gpu), 2)
    for f, args, kw in ((ck.rotary, (r, pos, q, k), dict(out=(k, q))), (ck.rotary, (r, pos, q, k), dict(out=(o, o))),
                        (ck.rotary, (r, pos, q, q), dict(out=(q, o))), (ck.rotary, (r, pos, q, q), dict(out=(o, q))),
                        (ck.kv_append, (cache, b, r, k, o), dict(q=q, out=k)), (ck.kv_append, (cache, b, r, o, k), dict(q=q, out=k))):
        with pytest.raises(ck.CkrError) as e:
            f(*args, **kw)
        assert e.value.code == ck.CKR_E_INVALID and "output" in str(e.value), str(e.value)
    torch.cuda.synchronize()


def test_no_heads_or_tokens_of_any_strides(gpu):
    r, pos = ck.Rotary(64), _i32([0, 1], gpu)
    q = torch.zeros(2, 2, 3, 64, device=gpu)
    for x, p in ((q[:, :, :0], pos), (q.transpose(1, 2)[:, :, :0], pos.new_zeros(3)), (q[:, :0], pos[:0]), (q[:0], pos)):
        assert ck.rotary(r, p, x).shape == x.shape
        a, b = ck.rotary(r, p, x, x)
        assert a.shape == b.shape == x.shape
    torch.cuda.synchronize()


def test_example_over_four_bits(gpu):
    """Tokens served over a parked and restored 4-bit cache."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "park_cache.py")
    spec = importlib.util.spec_from_file_location("park_cache", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(["--tokens", "6", "--layers", "1", "--bits", "4"]) == 0


def test_tensors_of_other_layouts(gpu):
    """Heads before tokens, positions of every other token, a rotary for another dtype: strides are followed."""
    r = ck.Rotary(64, interleaved=True)
    base = torch.randn(2, 6, 40, 64, device=gpu)                       # batch, heads, tokens, dim
    pos = _i32(np.arange(160).reshape(2, 80), gpu)[:, ::2]
    got = ck.rotary(r, pos, base.transpose(1, 2))
    want = ck.rotary(r, pos.contiguous(), base.transpose(1, 2).contiguous())
    assert torch.equal(got, want) and got.shape == (2, 40, 6, 64)
    shared = base[:, :1].expand(2, 6, 40, 64).transpose(1, 2)           # one head read by all
    assert torch.equal(ck.rotary(r, pos, shared), ck.rotary(r, pos, shared.contiguous()))
    x = base[:, :1].clone().requires_grad_()                            # the gradient of a broadcast input
    y = ck.rotary(r, pos, x.expand(2, 6, 40, 64).transpose(1, 2))
    g = torch.randn_like(y)
    d, = torch.autograd.grad(y, x, g)
    with torch.no_grad():
        back = ck.rotary(r, pos, g, inverse=True).transpose(1, 2).sum(1, keepdim=True)
    assert torch.allclose(d, back, rtol=0, atol=6 * 2 * ko.U32 * 6 * 8)   # six values of a few units, two orders of their sum
    odd = torch.randn(33 * 3 * 50 + 1, device=gpu)[1:].view(33, 3, 50)  # rows on 4-byte boundaries
    p = _i32(np.arange(33), gpu)
    assert torch.equal(ck.rotary(ck.Rotary(46), p, odd), ck.rotary(ck.Rotary(46), p, odd.clone()))


@pytest.mark.parametrize("rot,dim,inter", [(64, 128, False), (40, 80, False), (48, 64, True), (128, 128, False), (6, 32, False)])
@pytest.mark.parametrize("n", [1, 700])
def test_append_in_place_of_parts_of_heads(gpu, rot, dim, inter, n):
    """Queries turned in place, whose lanes read values that other lanes write; many tokens a block."""
    cache = ck.KvCache.empty(-(-n // 16), 16, 2, dim, ck.BF16)
    b = ck.KvBatch(_i32([range(-(-n // 16))], gpu), _i32([0], gpu), _i32([0, n], gpu), n)
    r = ck.Rotary(rot, interleaved=inter)
    x = torch.randn(n, 9, dim, device=gpu).to(torch.bfloat16)
    want = ck.rotary(r, _i32(range(n), gpu), x[:, :5].clone())
    wk = ck.rotary(r, _i32(range(n), gpu), x[:, 5:7].clone())
    v = x[:, 7:].clone()
    q = x[:, :5]
    assert ck.kv_append(cache, b, r, x[:, 5:7], x[:, 7:], q=q, out=q) is q
    assert torch.equal(q, want) and torch.equal(x[:, 7:], v)
    k2, v2 = ck.kv_read(cache, b)
    assert torch.equal(k2, wk) and torch.equal(v2, v)
