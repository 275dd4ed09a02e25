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


def test_pinning_takes_no_more_than_the_tensor(pkg, cuda):
    """Two tensors in one page, and what lies around them: only the tensors count as pinned, and both are read whole."""
    mc = pkg.moe_cache
    rt = torch.cuda.cudart()
    E, rows, K = 4, 8, 64
    n = E * rows * 68                                             # 2176 bytes of Q8_0: 34 per 32 values
    heap = torch.zeros(8 * 4096, dtype=torch.uint8)
    page = -heap.data_ptr() % 4096 + 4096
    starts = [page + 256, page + 256 + n + 16, page + 2 * 4096 + 3000 // 16 * 16]     # the last one in two pages
    rng = torch.Generator().manual_seed(1)
    mc.configure(enabled=True, slots=2, budget_gb=1.0)
    pinned = []
    try:
        tensors = []
        for i, at in enumerate(starts):
            view = heap[at: at + n].view(E, rows, 68)
            blocks = view.view(E, rows, 2, 34)
            blocks[..., :2] = torch.tensor([1.0], dtype=torch.float16).view(torch.uint8)        # scale 1, codes i8
            blocks[..., 2:] = torch.randint(-5, 6, (E, rows, 2, 32), generator=rng).to(torch.int8).view(torch.uint8)
            t = mc.expert_tensor(view, mc.Q8_0, K, rows, name=f"blk.{i}.ffn_up_exps.weight")
            assert not mc.wants(t) and mc.pin_host(t) and mc.pin_host(t) and mc.wants(t)
            pinned.append(view.data_ptr())
            tensors.append((t, view))
        held = torch.zeros(heap.numel(), dtype=torch.bool)
        for at in starts:
            held[at: at + n] = True
        for at in sorted({a + d for a in starts for d in (-1, 0, n - 1, n)} | {page, page + 4095, page + 4096, page + 3 * 4096 - 1}):
            probe = mc.expert_tensor(heap[at: at + 68].view(2, 1, 34), mc.Q8_0, 32, 1)       # (wants() asks about its first byte)
            assert mc.wants(probe) == bool(held[at]), at - page
        x = torch.ones((1, K), device=cuda)
        for t, view in tensors:
            want = view.view(E, rows, 2, 34)[..., 2:].view(torch.int8).float().sum((2, 3))
            for e in range(E):
                dst = torch.zeros((1, 1, rows), device=cuda)
                mc.mul_mat_vec_q(t, x, mc.F32, torch.full((1, 1), e, dtype=torch.int32, device=cuda), dst, ncols_dst=1, nchannels_y=1,
                                 nchannels_dst=1, stride_col_y=K, stride_col_dst=rows, stride_channel_y=K, stride_channel_dst=rows,
                                 ids_stride=1)
                # x is quantised to 127 steps of 1 / 127: its scale and the product round
                assert ((dst[0, 0].cpu() - want[e]).abs() <= 4 * 2.0 ** -11 * 5 * K).all()
        torch.cuda.synchronize()
        assert mc.device_error() == 0
    finally:
        torch.cuda.synchronize()
        mc.reset()
        for p in pinned:
            rt.cudaHostUnregister(p)


def test_a_tensor_that_is_pinned_in_part_is_refused(pkg, cuda):
    """Its first bytes answer for pinned memory, the others would be read from pageable memory."""
    mc = pkg.moe_cache
    rt = torch.cuda.cudart()
    heap = torch.zeros(4 * 4096, dtype=torch.uint8)
    at = -heap.data_ptr() % 4096 + 64
    mc.configure(enabled=True)
    try:
        for part in ((0, 512), (2176 - 512, 512)):
            p = heap.data_ptr() + at + part[0]
            assert int(rt.cudaHostRegister(p, part[1], 0)) == 0
            t = mc.expert_tensor(heap[at: at + 2176].view(4, 8, 68), mc.Q8_0, 64, 8, name="part")
            assert not mc.pin_host(t)
            rt.cudaHostUnregister(p)
    finally:
        mc.reset()
