"""Host memory that a caller registers: what lies beside it and what the heap makes of it later."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_enrolling_from_registered_heap_memory(pkg, cuda):
    """The first use of an expert tensor copies its table from memory that the heap gives back behind the call. Blocks of that
    size are registered and free before it, so that the heap may hand one out, and the stream is busy, so that a copy
    straight from one would read what comes to lie there: the table on the device has to be the tensor's."""
    mc = pkg.moe_cache
    rt, libc = torch.cuda.cudart(), ctypes.CDLL(None)
    libc.malloc.restype, libc.malloc.argtypes, libc.free.argtypes = ctypes.c_void_p, [ctypes.c_size_t], [ctypes.c_void_p]
    E, rows, K = 34, 8, 256
    sizes = (8 * E, 4 * E)                                # a table's bytes, a slot map's
    mc.configure(enabled=True, slots=4, budget_gb=1.0)
    held, registered = [], []
    try:
        w = torch.zeros((E, rows, 84), dtype=torch.uint8).pin_memory()
        t = mc.expert_tensor(w, mc.Q2_K, K, rows, name="blk.0.ffn_up_exps.weight")
        x = torch.zeros((1, K), device=cuda)
        ids, dst = torch.zeros((1, 1), dtype=torch.int32, device=cuda), torch.zeros((1, 1, rows), device=cuda)
        torch.cuda.synchronize()
        blocks = [(libc.malloc(n), n) for n in sizes for _ in range(7)]
        for p, n in blocks:
            if int(rt.cudaHostRegister(p, n, 0)) == 0:
                registered.append(p)
        assert len(registered) == len(blocks)
        for p, _ in blocks:
            libc.free(p)
        torch.cuda._sleep(20_000_000)                     # (a bounded spin of some milliseconds)
        mc.mul_mat_vec_q(t, x, mc.F32, ids, dst, ncols_dst=1, nchannels_y=1, nchannels_dst=1, stride_col_y=K, stride_col_dst=rows,
                         stride_channel_y=K, stride_channel_dst=rows, ids_stride=1)
        held = [(libc.malloc(n), n) for n in sizes for _ in range(14)]
        for p, n in held:
            ctypes.memset(p, 0, n)
        torch.cuda.synchronize()
        tbl, n_slots, _ = mc.table(t)
        assert n_slots == 4 and tbl == [-1] * E
        assert torch.equal(dst, torch.zeros_like(dst)) and mc.device_error() == 0
    finally:
        torch.cuda.synchronize()
        for p in registered:
            rt.cudaHostUnregister(p)
        for p, _ in held:
            libc.free(p)
        mc.reset()
