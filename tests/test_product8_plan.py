"""Which kernel makes a product of 8-bit tensors: host code that needs no device.  Whatever the sizes, and whatever a tuning build is told to do, the
kernel is one that takes them; and the sizes at which the GPU tests check a kernel are ones that go by it."""
import ctypes
import os
import random
import subprocess

import pytest

from savanna_amd import _lib

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")
TOKENS, TILE, TALL, WIDE = range(4)
ENTRY = """
#include "gcg_product8_plan.h"
extern "C" void plan(long long M, long long N, long long K, const char *kernel, const char *parts, long long *out)
{
    const gcg::Plan8 p = gcg::plan8(M, N, (int)((K + 127) / 128), kernel, parts);
    out[0] = p.kernel; out[1] = p.splits; out[2] = p.split_steps; out[3] = p.rest;
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    """(kernel, parts, blocks of a part, rows at the end by tiles of 256 x 128) of M, N, K and, in a tuning build, the kernel and parts asked for."""
    where = tmp_path_factory.mktemp("plan")
    (where / "plan.cpp").write_text(ENTRY)
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I" + CSRC, str(where / "plan.cpp"), "-o", str(where / "plan.so")], check=True)
    entry = ctypes.CDLL(str(where / "plan.so")).plan

    def plan(M, N, K, kernel=None, parts=None):
        out = (ctypes.c_longlong * 4)()
        text = lambda v: None if v is None else str(v).encode()                                     # noqa: E731
        entry(ctypes.c_longlong(M), ctypes.c_longlong(N), ctypes.c_longlong(K), text(kernel), text(parts), out)
        return tuple(out)
    return plan


def check(M, N, K, plan):
    kernel, parts, blocks, rest = plan
    what, steps = f"{M} x {N} x {K}: {plan}", (K + 127) // 128
    assert parts >= 1 and (parts - 1) * blocks < steps <= parts * blocks, what
    assert parts == 1 or blocks % 4 == 0, what                         # a part starts at a word of four scales
    assert rest == 0 or kernel == WIDE and parts == 1 and rest >= 256, what
    if kernel == TOKENS:                                               # sums of its own only, 32 blocks for each of eight or four waves
        assert parts == 1 and steps <= (256 if M <= 32 else 128), what
    elif kernel == TALL:
        assert M >= 256 and N >= 128, what
    elif kernel == WIDE:
        assert M - rest >= 256 and N >= 256, what
    else:
        assert kernel == TILE, what


def sizes(n, seed):
    rng = random.Random(seed)
    some = lambda top: int(2 ** rng.uniform(0, top))                   # noqa: E731
    return [(some(rng.choice([6, 9, 15])), some(15), some(rng.choice([10, 15, 22]))) for _ in range(n)]


def test_every_size_has_a_kernel_that_takes_it(plan):
    for M, N, K in sizes(4000, 1):
        check(M, N, K, plan(M, N, K))


def test_what_a_tuning_build_is_told_is_taken_where_the_kernel_takes_it(plan):
    for M, N, K in sizes(400, 2) + [(8, 4096, 4096), (1, 1, 1), (33, 5, 20000), (64, 300, 16384), (65, 300, 16384), (255, 256, 512), (256, 127, 512)]:
        for kernel in (-1, 0, 1, 2, 3, 4, "x", ""):
            for parts in (None, -3, 0, 1, 2, 3, 7, 32, 1000, "x"):
                check(M, N, K, plan(M, N, K, kernel, parts))
    assert plan(4096, 4096, 4096, WIDE, 2)[:2] == (WIDE, 2) and plan(8, 4096, 4096, TILE, 4)[:2] == (TILE, 4) and plan(100, 512, 512, TOKENS)[0] == TOKENS
