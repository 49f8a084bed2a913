"""The C header as programs in C and C++ include it."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
#include "checkers_amd.h"
/* a cache's scales are floats, the powers of a 4-bit cache bytes in their place */
float* scales(ckr_kv_cache* c, float* s) { c->d_v_scale = s; return c->d_k_scale; }
uint8_t* powers(ckr_kv_cache* c, uint8_t* p) { c->d_v_power = p; return c->d_k_power; }
int main(void) {
    float s[2];
    ckr_kv_cache c = {0};
    c.d_k_scale = s, c.d_v_scale = s + 1;
    return sizeof c == 136 && (void*)c.d_k_power == (void*)s && scales(&c, s + 1) == s ? 0 : 1;
}
"""


@pytest.mark.parametrize("compiler,flags,suffix", [("gcc", ["-std=c11"], "c"), ("gcc", [], "c"), ("g++", ["-std=c++11"], "cpp"), ("g++", ["-std=c++17"], "cpp")])
def test_scales_of_a_cache(tmp_path, compiler, flags, suffix):
    src, exe = tmp_path / f"program.{suffix}", tmp_path / "program"
    src.write_text(PROGRAM)
    subprocess.run([compiler, *flags, "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    subprocess.run([str(exe)], check=True)
