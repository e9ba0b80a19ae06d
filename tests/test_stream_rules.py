"""The rules by which the stream operators' launchers choose (csrc/kernels.h), compiled and run on the host."""
import subprocess

from conftest import ROOT

PROGRAM = r"""
#include <cstdio>
#include <cstdlib>

#include "kernels.h"

#define CHECK(c) do { if (!(c)) { std::printf("line %d: %s\n", __LINE__, #c); std::exit(1); } } while (0)

int main() {
    static float x[4], y[4];
    auto call = [&](const float *q, float *q_out, int heads, int kv_heads, long tokens) {
        vh::CacheRows a{};
        a.q = q;
        a.q_out = q_out;
        a.k = a.v = kv_heads ? x : nullptr;
        a.heads = heads;
        a.kv_heads = kv_heads;
        a.tokens = (int)tokens;
        a.head_dim = 48;
        return vh::rows_pass_caches(a);
    };
    const long at = (64l << 20) / (24 * 48 * 4);  // tokens that stay below, and one more
    CHECK(at == 14563);
    // K and V alone (no Q, so no pointers to one): three times as much.
    CHECK(!call(nullptr, nullptr, 0, 12, 3 * at) && call(nullptr, nullptr, 0, 12, 3 * (at + 1)));
    // From QKV rows, and a rotation into another tensor.
    CHECK(!call(x, y, 16, 4, at) && call(x, y, 16, 4, at + 1) && !call(x, y, 24, 0, at) && call(x, y, 24, 0, at + 1));
    // A rotation in place: four times as much.
    CHECK(!call(x, x, 24, 0, at + 1) && !call(x, x, 24, 0, 4 * at) && call(x, x, 24, 0, 4 * (at + 1)));
    CHECK(call(x, y, 65535, 65535, 1 << 27));  // past 32 bits
}
"""


def test_calls_that_pass_by_the_caches(tmp_path):
    src, exe = tmp_path / "rules.cpp", tmp_path / "rules"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    f"-I{ROOT / 'vestra-kernels_amd' / 'csrc'}", "-o", exe, src], check=True)
    run = subprocess.run([exe], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout
