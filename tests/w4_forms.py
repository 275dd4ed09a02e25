"""Products with 4-bit matrices whose sizes make the plan take each of its forms: 8 or 16 MMA columns, K in one piece or
shared by a cluster of 2 or 4, in one pass or several, with ids or one matrix, with a gate or without."""
import ctypes
from importlib import import_module

TYPES = {"f32": 0, "f16": 1, "bf16": 30}

# (tiles of 8 columns, CTAs of a cluster, several passes), rows, K, group, zeros, type of x, tokens, matrices, picks (0:
# one matrix, no ids), gate
CASES = [
    ((1, 1, False), 768, 2048, 32, True, "bf16", 1, 1, 0, False),
    ((1, 1, False), 1000, 2000, 64, True, "f16", 1, 1, 0, False),
    ((1, 1, False), 1024, 2048, 128, False, "f32", 1, 1, 0, True),
    ((1, 1, False), 768, 2048, 128, True, "bf16", 1, 1, 0, True),
    ((1, 1, False), 1000, 2000, 256, False, "f16", 1, 8, 2, False),
    ((1, 1, False), 1024, 2048, 32, True, "f32", 1, 8, 2, False),
    ((1, 1, False), 768, 2048, 64, True, "bf16", 1, 8, 2, True),
    ((1, 1, False), 1000, 2000, 128, False, "f16", 1, 8, 2, True),
    ((1, 1, True), 1024, 8192, 128, True, "f32", 40, 8, 2, False),
    ((1, 1, True), 1000, 8100, 256, False, "f32", 32, 8, 2, False),
    ((1, 1, True), 500, 16300, 32, True, "bf16", 16, 24, 4, True),
    ((1, 1, True), 512, 16384, 64, True, "f16", 16, 24, 4, True),
    ((1, 2, False), 1024, 8192, 128, False, "bf16", 8, 1, 0, False),
    ((1, 2, False), 1000, 8100, 128, True, "f16", 8, 1, 0, False),
    ((1, 2, False), 1024, 8192, 256, False, "bf16", 2, 1, 0, True),
    ((1, 2, False), 1000, 8100, 32, True, "f16", 2, 1, 0, True),
    ((1, 2, False), 500, 16300, 64, True, "bf16", 2, 8, 2, False),
    ((1, 2, False), 512, 16384, 128, False, "f16", 2, 8, 2, False),
    ((1, 2, False), 500, 16300, 128, True, "bf16", 2, 8, 2, True),
    ((1, 2, False), 512, 16384, 256, False, "f16", 2, 8, 2, True),
    ((1, 2, True), 500, 16300, 32, True, "f32", 33, 1, 0, False),
    ((1, 2, True), 512, 16384, 64, True, "f32", 33, 1, 0, False),
    ((1, 2, True), 256, 32768, 128, False, "f32", 5, 8, 2, False),
    ((1, 2, True), 256, 32768, 128, True, "f32", 5, 8, 2, False),
    ((1, 2, True), 256, 32768, 256, False, "f32", 5, 8, 2, True),
    ((1, 2, True), 256, 32768, 128, False, "bf16", 8, 8, 2, True),
    ((1, 4, False), 500, 16300, 32, True, "f16", 1, 1, 0, False),
    ((1, 4, False), 256, 32768, 64, True, "bf16", 1, 1, 0, False),
    ((1, 4, False), 512, 16384, 128, True, "f16", 1, 1, 0, True),
    ((1, 4, False), 500, 16300, 256, False, "f32", 1, 1, 0, True),
    ((1, 4, False), 256, 32768, 32, True, "bf16", 1, 8, 2, False),
    ((1, 4, False), 512, 16384, 64, True, "f16", 1, 8, 2, False),
    ((1, 4, False), 500, 16300, 128, False, "f32", 1, 8, 2, True),
    ((1, 4, False), 256, 32768, 128, True, "bf16", 1, 8, 2, True),
    ((1, 4, True), 256, 32768, 256, False, "f32", 4, 1, 0, False),
    ((1, 4, True), 256, 32768, 32, True, "f16", 8, 1, 0, False),
    ((1, 4, True), 256, 32768, 64, True, "f32", 3, 1, 0, True),
    ((1, 4, True), 256, 32768, 128, False, "bf16", 8, 1, 0, True),
    ((1, 4, True), 256, 32768, 128, True, "f16", 4, 8, 2, False),
    ((1, 4, True), 256, 32768, 256, False, "f32", 2, 8, 2, False),
    ((1, 4, True), 256, 32768, 32, True, "bf16", 3, 8, 2, True),
    ((1, 4, True), 256, 32768, 64, True, "f16", 3, 8, 2, True),
    ((2, 1, False), 2048, 2048, 128, False, "f32", 5, 1, 0, False),
    ((2, 1, False), 2048, 2048, 128, True, "bf16", 11, 1, 0, False),
    ((2, 1, False), 2048, 2048, 256, False, "f16", 11, 1, 0, True),
    ((2, 1, False), 768, 2048, 32, True, "f32", 16, 1, 0, True),
    ((2, 1, False), 768, 2048, 64, True, "bf16", 16, 8, 2, False),
    ((2, 1, False), 768, 2048, 128, False, "f16", 16, 8, 2, False),
    ((2, 1, False), 1024, 2048, 128, True, "f32", 8, 8, 2, True),
    ((2, 1, False), 768, 2048, 256, False, "bf16", 16, 8, 2, True),
    ((2, 1, True), 11008, 4096, 32, True, "f16", 16, 1, 0, False),
    ((2, 1, True), 4096, 4096, 64, True, "f32", 32, 1, 0, False),
    ((2, 1, True), 4000, 4100, 128, False, "bf16", 100, 1, 0, True),
    ((2, 1, True), 4096, 4096, 128, True, "f16", 64, 1, 0, True),
    ((2, 1, True), 4000, 4100, 256, False, "f32", 8, 8, 2, False),
    ((2, 1, True), 4000, 4100, 32, True, "bf16", 16, 8, 2, False),
    ((2, 1, True), 4096, 4096, 64, True, "f16", 16, 8, 2, True),
    ((2, 1, True), 4000, 4100, 128, False, "f32", 8, 8, 2, True),
    ((2, 2, False), 1000, 8100, 128, True, "bf16", 11, 1, 0, False),
    ((2, 2, False), 1024, 8192, 256, False, "f16", 11, 1, 0, False),
    ((2, 2, False), 4096, 4096, 32, True, "f32", 8, 1, 0, True),
    ((2, 2, False), 4000, 4100, 64, True, "bf16", 16, 1, 0, True),
    ((2, 2, False), 512, 16384, 128, False, "f16", 3, 8, 2, False),
    ((2, 2, False), 500, 16300, 128, True, "bf16", 3, 8, 2, False),
    ((2, 2, False), 512, 16384, 128, False, "f16", 3, 8, 2, True),
    ((2, 2, False), 500, 16300, 128, True, "bf16", 3, 8, 2, True),
    ((2, 2, True), 1000, 8100, 256, False, "f32", 100, 1, 0, False),
    ((2, 2, True), 1024, 8192, 32, True, "f32", 100, 1, 0, False),
    ((2, 2, True), 1000, 8100, 64, True, "f32", 100, 1, 0, True),
    ((2, 2, True), 1024, 8192, 256, False, "f32", 100, 1, 0, True),
    ((2, 2, True), 1000, 8100, 32, True, "f16", 16, 8, 2, False),
    ((2, 2, True), 1024, 8192, 64, True, "bf16", 16, 8, 2, False),
    ((2, 2, True), 512, 16384, 128, False, "f16", 16, 8, 2, True),
    ((2, 2, True), 500, 16300, 128, True, "bf16", 16, 8, 2, True),
    ((2, 4, False), 512, 16384, 256, False, "f16", 11, 1, 0, False),
    ((2, 4, False), 1000, 8100, 32, True, "f32", 5, 1, 0, False),
    ((2, 4, False), 500, 16300, 64, True, "bf16", 11, 1, 0, True),
    ((2, 4, False), 512, 16384, 128, False, "f16", 11, 1, 0, True),
    ((2, 4, False), 256, 32768, 128, True, "bf16", 3, 8, 2, False),
    ((2, 4, False), 256, 32768, 128, False, "f16", 3, 8, 2, False),
    ((2, 4, False), 256, 32768, 128, True, "bf16", 3, 8, 2, True),
    ((2, 4, False), 256, 32768, 128, False, "f16", 3, 8, 2, True),
    ((2, 4, True), 500, 16300, 256, False, "f32", 24, 1, 0, False),
    ((2, 4, True), 512, 16384, 32, True, "f32", 24, 1, 0, False),
    ((2, 4, True), 500, 16300, 64, True, "f32", 24, 1, 0, True),
    ((2, 4, True), 512, 16384, 256, False, "bf16", 33, 1, 0, True),
    ((2, 4, True), 500, 16300, 32, True, "f16", 32, 8, 2, False),
    ((2, 4, True), 512, 16384, 64, True, "f32", 24, 8, 2, False),
    ((2, 4, True), 500, 16300, 128, True, "bf16", 32, 8, 2, True),
    ((2, 4, True), 512, 16384, 256, False, "f16", 32, 8, 2, True),
]


B200 = (148, 74, 33)      # CTAs, clusters of 2 and of 4 that run at once


def plan(pkg, rows, K, group, zeros, dtype, n, E, k, gate, slots=None):
    """By the device's slots where they are not given: [tiles of 8 columns, CTAs of a cluster, warps that share K, row tiles of a block, passes, whether x is staged first]"""
    lm = import_module("a6000-custom-kernels_b200._lib")
    w, out = lm.MoeW4(None, E, rows, K, group, 1, zeros), (ctypes.c_int32 * 6)()
    slots = None if slots is None else (ctypes.c_int32 * 3)(*slots)
    lm.check(pkg.lib().moe_b200_w4_plan(ctypes.byref(w), gate, n, k, TYPES[dtype], slots, out))
    return list(out)


def form(pkg, case, slots=None):
    p = plan(pkg, *case[1:], slots)
    return p[0], p[1], p[4] > 1
