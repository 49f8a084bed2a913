"""add_rms_norm against 64 bits: the residual sum bit for bit, scales and values
within bounds derived from the arithmetic."""
import pytest
import torch

import checkers_amd as ck
from tests import kv_oracle as ko

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TAGS = {"bf16": ck.BF16, "f16": ck.F16, "f32": ck.F32, "f8": ck.F8, "i8": ck.I8}
# the sum of squares: at most 64 terms in a thread's order, then at most 6 + 16
# partial sums, so 86 roundings (43 after the root), and 8 more in the mean, the
# root, the reciprocal and the two products
REL = 51 * 2.0 ** -24


def _check(x, r, w, eps, out, scales, total, fmt, group):
    h, y = ko.norm(x.cpu(), None if r is None else r.cpu(), w.cpu(), eps)
    h32 = x.cpu().float() + (0 if r is None else r.cpu().float())
    assert torch.equal(total.cpu(), h32.to(x.dtype))
    out = out.cpu()
    if fmt in TYPES:
        bound = y.abs() * (ko.UNIT[out.dtype] + 2 * REL) + (2.0 ** -25 if fmt == "f16" else 2.0 ** -130)
        assert ((out.double() - y).abs() <= bound).all()
        return
    n = y.shape[1]
    parts = y.view(y.shape[0], -1, group or n)
    top = parts.abs().amax(-1)
    s = scales.cpu().double().view(top.shape)
    zero = top < 2.0 ** -100
    assert (s[zero] == 0).all()
    assert ((s - top / ko.TOP[fmt]).abs() <= (REL + 2.0 ** -23) * top / ko.TOP[fmt])[~zero].all()
    got = out.float().double().view(parts.shape) * s[..., None]
    # half a step of the code: of 1 in int8; in e4m3 2^-4 of the value, 2^-10 near zero
    step = 0.5 * s[..., None] if fmt == "i8" else torch.maximum(parts.abs() * 2.0 ** -4, 2.0 ** -10 * s[..., None])
    assert ((got - parts).abs() <= step * (1 + 2.0 ** -10) + parts.abs() * 4 * REL)[~zero].all()
    assert (out.float().view(parts.shape)[zero] == 0).all()


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,n", [(1, 4096), (3, 1), (5, 7), (2, 64), (4, 511), (3, 520), (2, 2048), (3, 2056), (1, 5120),
                                    (2, 8192), (3, 8193), (2, 12000), (1, 20_000), (2, 40_001), (1, 65_536)])
def test_norm(gpu, typ, rows, n):
    g = torch.Generator(device=gpu).manual_seed(n)
    t = TYPES[typ]
    x, r = ((torch.randn(rows, n, generator=g, device=gpu) * s).to(t) for s in (1.0, 3.0))
    w = (1 + 0.2 * torch.randn(n, generator=g, device=gpu))
    for fmt in (typ, "f8", "i8"):
        for group in (0, 32, 128, 256) if fmt in ko.TOP else (0,):
            if group and n % group:
                continue
            for res, wt in ((r, w.to(t)), (None, w)):
                print(f"[case] norm {typ} {rows}x{n} -> {fmt} group={group} residual={res is not None}", flush=True)
                out, scales, total = ck.add_rms_norm(x, res, wt, 1e-5, TAGS[fmt], group=group)
                torch.cuda.synchronize()
                _check(x, res, wt, 1e-5, out, scales, total, fmt, group)


@pytest.mark.parametrize("typ", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,n", [(33, 8), (17, 100), (16, 128), (15, 129), (9, 256), (7, 257), (6, 768), (5, 1024), (7, 1500)])
def test_norm_of_short_rows(gpu, typ, rows, n):
    """Rows that share a block, the last block partly filled."""
    t = TYPES[typ]
    x, r = ((torch.randn(rows, n, device=gpu) * s).to(t) for s in (1.0, 3.0))
    w = torch.randn(n, device=gpu).to(t)
    for fmt, group in ((typ, 0), ("f8", 0), ("i8", 0), ("f8", 32), ("i8", 64), ("f8", 128), ("i8", 256)):
        if group and n % group:
            continue
        print(f"[case] norm short {typ} {rows}x{n} -> {fmt} group={group}", flush=True)
        out, scales, total = ck.add_rms_norm(x, r, w, 1e-5, TAGS[fmt], group=group)
        torch.cuda.synchronize()
        _check(x, r, w, 1e-5, out, scales, total, fmt, group)


@pytest.mark.parametrize("typ", ["bf16", "f32"])
def test_norm_strides_and_alignment(gpu, typ):
    """Rows inside wider ones, starting at odd elements; outputs likewise."""
    t, n = TYPES[typ], 1056
    for first, stride in ((0, n + 8), (1, n + 3), (4, n + 64)):
        print(f"[case] norm strides {typ} {first} {stride}", flush=True)
        big = torch.randn(6, 4 * stride + 9, device=gpu).to(t)
        x, r = (torch.as_strided(big, (5, n), (stride, 1), first + k) for k in (0, 2))
        w = torch.randn(n + 9, device=gpu).to(t)[first:first + n]
        for fmt, group in ((typ, 0), ("f8", 32), ("i8", 0)):
            o = torch.zeros(5 * stride + 9, dtype=torch.uint8, device=gpu).view(torch.int8) if fmt != typ else torch.zeros(5 * stride + 9, dtype=t, device=gpu)
            o = o.view(torch.float8_e4m3fn) if fmt == "f8" else o
            out = torch.as_strided(o, (5, n), (stride, 1), first)
            tot = torch.as_strided(torch.zeros(5 * stride + 9, device=gpu).to(t), (5, n), (stride, 1), first)
            out, scales, tot = ck.add_rms_norm(x, r, w, 1e-6, TAGS[fmt], group=group, out=out, total=tot)
            torch.cuda.synchronize()
            _check(x, r, w, 1e-6, out.contiguous() if fmt != "f8" else out.view(torch.uint8).contiguous().view(torch.float8_e4m3fn),
                   scales, tot.contiguous(), fmt, group)


@pytest.mark.parametrize("which", ["x", "residual"])
def test_norm_in_place(gpu, which):
    x, r = (torch.randn(9, 4096, device=gpu).half() for _ in range(2))
    w = torch.ones(4096, device=gpu).half()
    a, b = x.clone(), r.clone()
    out, scales, total = ck.add_rms_norm(a, b, w, 1e-5, ck.F8, total=a if which == "x" else b)
    torch.cuda.synchronize()
    _check(x, r, w, 1e-5, out, scales, total, "f8", 0)


def test_norm_of_empty_zero_and_non_finite_rows(gpu):
    x = torch.randn(6, 512, device=gpu)
    x[0] = 0
    x[1, 5] = float("inf")
    x[2, 500] = float("nan")
    x[3] *= 1e-30
    w = torch.ones(512, device=gpu)
    for fmt in ("f8", "i8"):
        for group in (0, 64):
            out, scales, total = ck.add_rms_norm(x, None, w, 1e-5, TAGS[fmt], group=group)
            s, o = scales.view(6, -1).cpu(), out.float().cpu()
            assert (s[0] == 0).all() and (o[0] == 0).all()
            assert torch.isnan(s[2]).all() and (o[2] == 0).all()
            # an infinity: h / rms is NaN there and 0 elsewhere
            assert torch.isnan(s[1, 0]) and (o[1] == 0).all()
            keep = torch.tensor([3, 4, 5], device=gpu)
            _check(x[keep], None, w, 1e-5, out.view(torch.uint8)[keep].view(out.dtype), scales[keep], total[keep], fmt, group)
    out, scales, total = ck.add_rms_norm(torch.zeros(0, 512, device=gpu), None, w, 1e-5, ck.F8)
    assert out.shape == (0, 512) and scales.shape == (0,)


def test_norm_in_a_graph_and_on_a_stream(gpu):
    x, r = (torch.randn(7, 1024, device=gpu).to(torch.bfloat16) for _ in range(2))
    w = torch.randn(1024, device=gpu).to(torch.bfloat16)
    bufs = ck.add_rms_norm(x, r, w, 1e-5, ck.F8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    other = ck.add_rms_norm(x, r, w, 1e-5, ck.F8, stream=side)
    side.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(bufs, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ck.add_rms_norm(x, r, w, 1e-5, ck.F8, out=bufs[0], scales=bufs[1], total=bufs[2])
    for i in range(4):
        x.copy_(torch.randn(7, 1024, device=gpu))
        graph.replay()
        torch.cuda.synchronize()
        want = ck.add_rms_norm(x, r, w, 1e-5, ck.F8)
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(bufs, want)), i


def test_norm_refusals(gpu):
    x = torch.zeros(2, 96, device=gpu).half()
    w = torch.zeros(96, device=gpu).half()

    def bad(part, *a, **kw):
        with pytest.raises(ck.CkrError) as e:
            ck.add_rms_norm(*a, **kw)
        assert e.value.code == ck.CKR_E_INVALID and part in str(e.value), str(e.value)

    bad("group", x, None, w, 1e-5, ck.F8, group=64)
    bad("group", x, None, w, 1e-5, ck.F8, group=48)
    bad("group", x, None, w, 1e-5, group=32)
    bad("weight", x, None, w[:90], 1e-5)
    bad("weight", x, None, w.to(torch.bfloat16), 1e-5)
    bad("eps", x, None, w, -1.0)
    bad("eps", x, None, w, float("nan"))
    bad("type", x, x.float(), w)
    bad("type", x.int(), None, w)
    bad("output", x, None, w, 1e-5, ck.F32)
    bad("scales", x, None, w, 1e-5, ck.F8, scales=torch.zeros(3, device=gpu))
    bad("[2, 96]", x, x[:1], w)
    bad("[2, 96]", x.t().contiguous().t(), None, w)
    bad("65536", torch.zeros(1, 65_544, device=gpu), None, torch.zeros(65_544, device=gpu))
    bad("GPU", x.cpu(), None, w)


def test_norm_refuses_to_lose_a_gradient(gpu):
    """Tensors that require gradients: refused where gradients are recorded, taken where not."""
    x, r = (torch.randn(3, 64, device=gpu) for _ in range(2))
    w = torch.ones(64, device=gpu)
    want = ck.add_rms_norm(x, r, w)
    for i in range(3):
        t = [x, r, w]
        t[i] = t[i].clone().requires_grad_()
        with pytest.raises(ck.CkrError) as e:
            ck.add_rms_norm(*t)
        assert e.value.code == ck.CKR_E_INVALID and "no backward" in str(e.value)
        with torch.no_grad():
            got = ck.add_rms_norm(*t)
        again = ck.add_rms_norm(*(y.detach() for y in t))
        assert torch.equal(got[0], want[0]) and torch.equal(again[2], want[2])
