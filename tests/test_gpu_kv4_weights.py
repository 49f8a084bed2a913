"""How many bits of the weights attention over a cache in 4 bits keeps, by its error against
64 bits beside that of rounding the exact result once."""
import numpy as np
import pytest
import torch

import checkers_amd as ck
from tests import kv4_oracle as k4
from tests import kv_oracle as ko
from tests.test_gpu_kv4 import TYPES, _attend, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("typ,group,dim,old,chunk", [
    ("f16", 4, 128, 300, 3), ("f16", 4, 64, 90, 10),                               # few rows
    ("f16", 4, 128, 200, 30), ("f16", 2, 64, 100, 50), ("f16", 4, 256, 50, 40),    # up to 128
    ("f16", 4, 128, 200, 90), ("f16", 8, 64, 0, 100), ("f16", 4, 96, 300, 60),     # more
    ("bf16", 4, 128, 200, 30), ("bf16", 4, 128, 200, 90), ("bf16", 4, 128, 300, 3)])
def test_error_is_that_of_the_outputs_rounding(gpu, typ, group, dim, old, chunk):
    """A result off by d (relative, at random) before its rounding, which is off by r, is off by
    sqrt(r^2 + d^2): r is 0.29 steps' worth, about 2^-12.3 in float16 and 2^-9.3 in bfloat16.  Weights of
    16 bits and more have d < 2^-16, a factor of 1.003; of 11 bits d of 2^-12.5 or so, 1.3 in
    float16 and 1.01 in bfloat16.  Allowed: 1.05."""
    print(f"[case] {typ} {group} {dim} {old} {chunk}", flush=True)
    sq, cache, b, q, plan, out, lse = _attend(gpu, typ, 2, group, dim, 16, [old], [chunk], 0)
    k, v = (k4.as_numpy(_values(cache, n)) for n in ("k", "v"))
    ref = ko.attention(sq, k, v, q.cpu().double().numpy(), group, dim ** -0.5, 0)[0]
    once = torch.from_numpy(ref).to(TYPES[typ]).double().numpy()
    got = out.cpu().double().numpy()
    rms = lambda x: float(np.sqrt((x * x).mean()))
    print(f"  {rms(got - ref) / rms(once - ref):.4f}", flush=True)
    assert rms(got - ref) <= 1.05 * rms(once - ref)
