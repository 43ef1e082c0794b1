"""Which kernel takes a product of 8-bit codes, without a GPU: the sizes that the GPU tests run reach every kernel and number of
parts, and no size within the limits makes a launch that the GPU does not hold."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

from _i8plans import FEW, PLANS, TILE64, TILE128, TILE128X2, TILE256
from conftest import ROOT
from inferno_hip import _lib as L

TILE = {TILE64: 64, TILE128: 128, TILE128X2: 128, TILE256: 256}
MAIN = r"""
#include <stdio.h>
#include "gemm8_plan.h"
int main() {
    for (int m, n, k, accum; scanf("%d %d %d %d", &m, &n, &k, &accum) == 4;) {
        const Gemm8Plan p = gemm8_plan(m, n, k, accum);
        printf("%d %d\n", p.shape, p.parts);
    }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """The planner, compiled for the host: (m, n, k, accum) of many products to their kernels and parts."""
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run([cxx, "-O2", "-std=c++17", "-I", os.path.join(ROOT, "inferno.jl_amd", "csrc"), "-o", str(d / "plan"),
                    str(d / "main.cpp")], check=True)

    def ask(sizes):
        text = "".join("%d %d %d %d\n" % tuple(s) for s in sizes)
        out = subprocess.run([str(d / "plan")], input=text, capture_output=True, text=True, check=True).stdout
        got = [tuple(map(int, line.split())) for line in out.splitlines()]
        assert len(got) == len(sizes)
        return got
    return ask


def test_products_of_the_gpu_tests(plan):
    """They go where the list says, so that a change of the planner cannot take a kernel out of the tests unseen."""
    want = [(kernel, parts) for *_, kernel, parts in PLANS]
    assert plan([p[:4] for p in PLANS]) == want
    parts = {kernel: {p for at, p in want if at == kernel} for kernel in (FEW, *TILE)}
    assert parts == {FEW: {1}, TILE64: {1, 2, 3, 4, 6, 8}, TILE128: {1, 2, 3, 4, 6, 8}, TILE128X2: {1, 3},
                     TILE256: {1, 2, 3, 4, 6, 8}}


def test_the_library_plans_alike():
    """Its workspaces are those of the listed parts."""
    lib, nb = L.load(), C.c_size_t()
    for m, n, k, accum, _, parts in PLANS:
        L.check(lib.ihip_gemm_i8_ws_bytes(m, n, k, 4 if accum else 0, C.byref(nb)))
        assert nb.value == (parts * m * ((n + 3) // 4 * 4) * 4 if parts > 1 else 0), (m, n, k)


def test_nothing_else_is_reached(plan):
    """Sizes spread over the range take no kernel and number of parts that the list has not."""
    r = random.Random(41)
    at = lambda most: int(2 ** r.uniform(0, most))  # noqa: E731
    sizes = [(at(12), at(15), 16 * at(12), r.random() < 0.5) for _ in range(60000)]
    assert set(plan(sizes)) <= {(kernel, parts) for *_, kernel, parts in PLANS}


def test_launches_at_the_limits(plan):
    """Below 2^32 threads, workgroups and values of a workspace within 32-bit numbers."""
    r = random.Random(42)
    near = lambda e: max(1, min(1 << 23, (1 << e) + r.choice((-1, 0, 1))))  # noqa: E731
    sizes = [(near(i), near(j), k, a) for i in range(24) for j in range(24) for k in (16, 128, 1024, 4096, 65536) for a in (0, 1)]
    sizes += [(int(2 ** r.uniform(0, 23)), int(2 ** r.uniform(0, 23)), 16 * int(2 ** r.uniform(0, 12)), 0) for _ in range(40000)]
    sizes += [(1 << 23, n, k, a) for n in range(8000, 8193) for k in (16, 64, 256) for a in (0, 1)]
    sizes = [s for s in sizes if s[0] * s[1] <= 1 << 36]
    for (m, n, k, _), (kernel, parts) in zip(sizes, plan(sizes)):
        wgs = -(-m // 16) * -(-n // 16) if kernel == FEW else -(-m // TILE[kernel]) * -(-n // TILE[kernel])
        assert wgs * (128 if kernel == FEW else 512) < 1 << 32, (m, n, k)
        assert parts == 1 or parts * m * ((n + 3) // 4) < 1 << 31, (m, n, k)


def test_rows_at_the_limits():
    """Rows of codes that a launch does not hold are refused by name, before any launch; those that it holds pass that check (and
    are refused for a stride here)."""
    lib, at = L.load(), (C.c_uint8 * 64)()
    p = (C.addressof(at) + 15) & ~15
    for m, k, fits in ((1 << 23, 7184, False), (1 << 23, 65536, False), (1 << 22, 16400, False), ((1 << 23) - 1, 7184, True),
                       (1 << 23, 7168, True), (1 << 23, 16, True), ((1 << 22) - 1, 65536, True), (4300000, 14400, True)):
        for act in (0, 1, 2):
            a = L.GemmInput(p, 4, act, None, 1e-6, None, 0, 0)
            assert lib.ihip_quantize_i8(C.byref(a), m, k, p, k, p, None) == -22
            assert (b"2^32 threads" in lib.ihip_last_error()) == (not fits), (m, k, lib.ihip_last_error())
            assert fits == (b"ldx=4" in lib.ihip_last_error())
            assert fits or m * k > (1 << 36) - (1 << 33)
