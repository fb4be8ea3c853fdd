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


# Sizes at which the GPU tests check a kernel: by 256 x 256, by 256 x 128, by both, by 128 x 128, by groups of 64 rows; parts of the blocks
PLANS = {
    (4096, 4096, 128): (WIDE, 1, False), (3841, 4096, 640): (WIDE, 1, False), (4090, 4094, 1000): (WIDE, 1, False), (8200, 6000, 1300): (WIDE, 1, False),
    (14673, 2327, 124): (WIDE, 1, False), (2357, 3272, 242): (WIDE, 1, False),
    (1716, 1227, 15532): (WIDE, 4, False), (1716, 1227, 15400): (WIDE, 4, False), (274, 4257, 13982): (WIDE, 7, False), (5149, 775, 16335): (WIDE, 2, False),
    (2930, 795, 21788): (WIDE, 4, False),
    (12000, 11500, 1300): (WIDE, 1, True), (5003, 7683, 1301): (WIDE, 1, True), (70000, 257, 1300): (WIDE, 1, True), (16700, 1025, 900): (WIDE, 1, True),
    (2048, 4096, 128): (TALL, 1, False), (1900, 3970, 1101): (TALL, 1, False), (7675, 2057, 766): (TALL, 1, False), (2040, 2048, 16384): (TALL, 2, False),
    (1300, 2000, 7001): (TALL, 2, False), (600, 600, 17000): (TALL, 12, False),
    (606, 11384, 1158): (TILE, 1, False), (150, 15000, 10000): (TILE, 2, False), (67, 14005, 6507): (TILE, 4, False), (200, 300, 20000): (TILE, 20, False),
    (65, 64, 100): (TOKENS, 1, False), (300, 200, 5000): (TOKENS, 1, False), (1000, 1000, 8200): (TOKENS, 1, False), (1100, 33, 2000): (TOKENS, 1, False),
    (1, 4097, 32768): (TOKENS, 1, False), (64, 9000, 16384): (TOKENS, 1, False),
}


@pytest.mark.parametrize("size", PLANS)
def test_sizes_go_by_the_kernel_that_they_check(plan, size):
    """A size that goes by another kernel after a change of the estimates leaves its kernel without this test: choose another one."""
    kernel, parts, _, rest = plan(*size)
    assert (kernel, parts, rest > 0) == PLANS[size]


def test_the_parts_of_wide_tiles_end_in_every_rest_of_their_loop(plan):
    ends = set()
    for (M, N, K), (kernel, parts, _) in PLANS.items():
        if kernel == WIDE and parts > 1:
            ends.add(((K + 127) // 128 - (parts - 1) * plan(M, N, K)[2]) % 4)
    assert ends == {0, 1, 2, 3}
