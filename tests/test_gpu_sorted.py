"""Tokens sorted by expert and back, with gradients, against the plain 64-bit
implementation (sorted_ref)."""
import numpy as np
import pytest
import torch

import sorted_ref as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def f64(t):
    return t.detach().double().cpu().numpy()


def draw_ids(rng, n, k, E, drop=0.0):
    ids = rng.integers(0, E, size=(n, k)).astype(np.int32)          # the same expert twice in a token, too
    ids[rng.random((n, k)) < drop] = -1
    return ids


def rand(rng, shape, dtype, cuda, scale=1.0):
    return torch.from_numpy((scale * rng.normal(size=shape)).astype(np.float32)).to(cuda).to(DT[dtype])


def check_order(order, ids, E):
    want = R.order(ids, E)
    for got, ref in zip((order.rows, order.positions, order.experts, order.offsets), want):
        assert got.dtype == torch.int32
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
    return want


@pytest.mark.parametrize("n,k,E,drop", [
    (0, 4, 8, 0.0), (1, 1, 1, 0.0), (1, 1, 7, 1.0), (1, 8, 64, 0.0), (3, 2, 5, 0.5), (33, 1, 3, 0.1), (77, 6, 160, 0.1),
    (512, 8, 64, 0.0), (513, 8, 64, 0.0),        # the last call of one CTA, the first of a cluster
    (700, 7, 1024, 0.2), (1000, 32, 3, 0.0), (4097, 9, 513, 0.3), (20000, 8, 256, 0.0), (5000, 3, 1, 0.9), (900, 6, 40, 1.0),
])
def test_order(pkg, cuda, n, k, E, drop):
    rng = np.random.default_rng(n * 31 + k)
    ids = draw_ids(rng, n, k, E, drop)
    order = pkg.sort_by_expert(torch.from_numpy(ids).to(cuda), E)
    check_order(order, ids, E)
    assert pkg.moe_cache.device_error() == 0


def test_order_of_one_expert_and_of_sorted_runs(pkg, cuda):
    """Every count in one place, and long equal runs."""
    for ids, E in ((np.full((3000, 4), 5, np.int32), 9), (np.sort(np.random.default_rng(0).integers(0, 17, (2500, 4)), axis=None)
                                                          .astype(np.int32).reshape(2500, 4)[::-1].copy(), 17)):
        check_order(pkg.sort_by_expert(torch.from_numpy(ids).to(cuda), E), ids, E)


def test_ids_of_a_wider_buffer_and_bad_ids(pkg, cuda):
    rng = np.random.default_rng(3)
    wide = draw_ids(rng, 600, 12, 20)
    t = torch.from_numpy(wide).to(cuda)
    check_order(pkg.sort_by_expert(t[:, 2:9], 20), wide[:, 2:9], 20)
    check_order(pkg.sort_by_expert(t[4:5, 2:9], 20), wide[4:5, 2:9], 20)
    assert pkg.moe_cache.device_error() == 0
    for bad in (20, -2, 2 ** 31 - 1, -2 ** 31):
        ids = draw_ids(rng, 50, 3, 20)
        ids[7, 1] = bad
        order = pkg.sort_by_expert(torch.from_numpy(ids).to(cuda), 20)
        assert pkg.moe_cache.device_error() == pkg.moe_cache.DERR_BAD_ID
        check_order(order, ids, 20)               # as an empty slot
    assert pkg.moe_cache.device_error() == 0


SHAPES = [(1, 1, 1, 1, 0.0), (1, 8, 64, 2048, 0.0), (2, 3, 4, 17, 0.4), (9, 9, 30, 130, 0.2), (77, 6, 160, 1442, 0.1),
          (40, 2, 3, 4, 0.0), (5, 20, 6, 5000, 0.3), (600, 8, 16, 256, 0.05), (6, 4, 5, 96, 1.0)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,E,H,drop", SHAPES)
def test_there_and_back(pkg, cuda, n, k, E, H, drop, dtype):
    rng = np.random.default_rng(n + H)
    ids = draw_ids(rng, n, k, E, drop)
    x, y, shared = (rand(rng, (m, H), dtype, cuda) for m in (n, n * k, n))
    w = torch.from_numpy(rng.random((n, k)).astype(np.float32)).to(cuda)
    rows, order = pkg.dispatch_sorted(x, torch.from_numpy(ids).to(cuda), E)
    ref_rows, pos, _, _ = check_order(order, ids, E)
    np.testing.assert_array_equal(f64(rows), R.gather(f64(x), ref_rows, k))
    assert rows.dtype == x.dtype
    y[int((pos >= 0).sum()):] = float("nan")                        # nothing reads behind the last row
    clean = np.nan_to_num(f64(y))
    for sh in (None, shared):
        out = pkg.combine_sorted(y, order, w, shared=sh)
        assert out.dtype == y.dtype
        s, mag = R.combine(clean, pos, f64(w), None if sh is None else f64(sh))
        assert (np.abs(f64(out) - s) <= R.combine_tol(s, mag, k, dtype)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,k,E,H,drop", SHAPES)
def test_gradients(pkg, cuda, n, k, E, H, drop, dtype):
    """Against the formulas, and against differences: what is differentiated is linear in each argument, so
    <d_out, f(a + v) - f(a)> = <gradient, v>."""
    rng = np.random.default_rng(2 * n + H)
    ids = draw_ids(rng, n, k, E, drop)
    x, y, shared, d_rows, d_out = (rand(rng, (m, H), dtype, cuda) for m in (n, n * k, n, n * k, n))
    w = torch.from_numpy(rng.normal(size=(n, k)).astype(np.float32)).to(cuda)
    leaves = [t.requires_grad_() for t in (x, y, w, shared)]
    rows, order = pkg.dispatch_sorted(x, torch.from_numpy(ids).to(cuda), E)
    out = pkg.combine_sorted(y, order, w, shared=shared)
    d_x, d_y, d_w, d_s = torch.autograd.grad([rows, out], leaves, [d_rows, d_out])
    ref_rows, pos, _, _ = R.order(ids, E)
    s, mag = R.combine(f64(d_rows), pos, None)
    assert (np.abs(f64(d_x) - s) <= R.combine_tol(s, mag, k, dtype)).all()
    live = ref_rows >= 0
    t = np.maximum(ref_rows, 0) // k
    want = np.where(live[:, None], f64(d_out)[t] * f64(w).reshape(-1)[np.maximum(ref_rows, 0)][:, None], 0.0)
    assert (np.abs(f64(d_y) - want) <= 1.01 * (2.0 ** -24 + R.HALF[dtype]) * np.abs(want) + R.TINY[dtype]).all()
    prod = f64(d_out)[:, None] * R.picks(f64(y), pos)
    assert (np.abs(f64(d_w) - prod.sum(2)) <= 1.01 * (H + 5) * 2.0 ** -24 * np.abs(prod).sum(2) + H * 2.0 ** -149).all()
    assert torch.equal(d_s, d_out)
    if dtype != "f32":
        return
    # differences: sums of n k H terms of the forward's and the gradients' rounding, both 2^-24 of their parts (2 k + 1
    # or H + 5 of them)
    for leaf, grad, f, d in ((x, d_x, lambda a: pkg.gather_sorted(a, order), d_rows), (y, d_y, lambda a: pkg.combine_sorted(a, order, w), d_out),
                             (w, d_w, lambda a: pkg.combine_sorted(y, order, a), d_out)):
        v = torch.from_numpy(rng.normal(size=tuple(leaf.shape)).astype(np.float32)).to(cuda)
        with torch.no_grad():
            a1 = leaf + v
            diff = f64(f(a1)) - f64(f(leaf))
            step = f64(a1) - f64(leaf)
        left, right = (f64(d) * diff).sum(), (f64(grad) * step).sum()
        parts = np.abs(f64(d)).max() * (np.abs(f64(f(leaf))).sum() + np.abs(f64(f(a1))).sum()) + np.abs(f64(grad) * step).sum() + \
            (np.abs(prod).sum() if leaf is w else 0.0) * np.abs(step).max() + \
            np.abs(f64(d)).max() * 8 * k * np.sqrt(n * k * H) * max(1.0, np.abs(f64(w)).max()) * 4
        assert abs(left - right) <= (2 * k + H + 8) * 2.0 ** -24 * parts + 1e-30


def test_rows_of_wider_buffers(pkg, cuda):
    rng = np.random.default_rng(5)
    n, k, E, H = 19, 3, 4, 64
    ids = torch.from_numpy(draw_ids(rng, n, k, E, 0.2)).to(cuda)
    w = torch.rand((n, k), device=cuda)
    for dtype in DT:
        for pad, at in ((16, 0), (2, 1), (3, 0), (5, 3)):          # 16-, 4-, 2-byte aligned rows
            big = rand(rng, (n * k, H + pad), dtype, cuda)
            x, y, sh = big[:n, at:at + H], big[:, at:at + H], big[:n, at:at + H]
            rows, order = pkg.dispatch_sorted(x, ids, E)
            plain, _ = pkg.dispatch_sorted(x.contiguous(), ids, E)
            assert torch.equal(rows, plain)
            assert torch.equal(pkg.combine_sorted(y, order, w, shared=sh),
                               pkg.combine_sorted(y.contiguous(), order, w, shared=sh.contiguous()))
            yl = y.detach().requires_grad_()
            g = rand(rng, (n, H + pad), dtype, cuda)[:, at:at + H]
            wl = w.clone().requires_grad_()
            a = torch.autograd.grad(pkg.combine_sorted(yl, order, wl), [yl, wl], g)
            yc = y.contiguous().requires_grad_()
            b = torch.autograd.grad(pkg.combine_sorted(yc, order, wl), [yc, wl], g.contiguous())
            assert torch.equal(a[0], b[0])
            # d_weights are sums of H products whose order goes with the width of the loads: each order is within
            # (H + 5) 2^-24 of the products' magnitudes of the true sum (as in test_gradients), so two of them within twice that
            mag = np.abs(f64(g)[:, None] * R.picks(f64(y), order.positions.cpu().numpy())).sum(2)
            assert (np.abs(f64(a[1]) - f64(b[1])) <= 2.02 * (H + 5) * 2.0 ** -24 * mag).all()


def test_gradients_of_some_inputs(pkg, cuda):
    """Each leaf alone, an expanded gradient (of a sum), and no graph where none is asked for."""
    rng = np.random.default_rng(6)
    n, k, E, H = 21, 4, 6, 40
    ids = torch.from_numpy(draw_ids(rng, n, k, E, 0.2)).to(cuda)
    x, y, sh = (rand(rng, (m, H), "f32", cuda) for m in (n, n * k, n))
    w = torch.rand((n, k), device=cuda)
    rows, order = pkg.dispatch_sorted(x, ids, E)
    assert not rows.requires_grad
    args = {"y": y, "weights": w, "shared": sh}
    full = {a: t.clone().requires_grad_() for a, t in args.items()}
    pkg.combine_sorted(full["y"], order, full["weights"], shared=full["shared"]).sum().backward()
    for name in args:
        one = {a: t.clone().requires_grad_(a == name) for a, t in args.items()}
        pkg.combine_sorted(one["y"], order, one["weights"], shared=one["shared"]).sum().backward()
        assert torch.equal(one[name].grad, full[name].grad)
        assert all(one[a].grad is None for a in args if a != name)
    xl = x.clone().requires_grad_()
    pkg.gather_sorted(xl, order).sum().backward()
    live = (order.positions >= 0).sum(1, keepdim=True).float()
    assert torch.equal(xl.grad, live.expand(n, H))
    with torch.no_grad():
        assert not pkg.combine_sorted(full["y"], order, full["weights"]).requires_grad
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(pkg.gather_sorted(xl, order).sum(), xl, create_graph=True)
        g.sum().backward()


def test_dropped_picks_keep_nans_out(pkg, cuda):
    """A weight, a row or a gradient that belongs to no sorted row reaches nothing."""
    rng = np.random.default_rng(7)
    n, k, E, H = 12, 3, 4, 32
    ids = draw_ids(rng, n, k, E, 0.4)
    order = pkg.sort_by_expert(torch.from_numpy(ids).to(cuda), E)
    w = torch.rand((n, k), device=cuda)
    w[order.positions < 0] = float("nan")
    live = int((ids >= 0).sum())
    y = torch.randn((n * k, H), device=cuda)
    y[live:] = float("inf")
    y.requires_grad_()
    w.requires_grad_()
    out = pkg.combine_sorted(y, order, w)
    assert torch.isfinite(out).all()
    d_y, d_w = torch.autograd.grad(out, [y, w], torch.randn_like(out))
    assert torch.isfinite(d_y).all() and torch.isfinite(d_w).all()
    assert (d_w[order.positions < 0] == 0).all() and (d_y[live:] == 0).all()


def test_streams_graphs_and_backward_in_a_graph(pkg, cuda):
    rng = np.random.default_rng(8)
    n, k, E, H = 300, 4, 12, 200
    ids = torch.from_numpy(draw_ids(rng, n, k, E, 0.1)).to(cuda)
    x, y = (rand(rng, (m, H), "bf16", cuda).requires_grad_() for m in (n, n * k))
    w = torch.rand((n, k), device=cuda).requires_grad_()
    d_rows, d_out = (rand(rng, (m, H), "bf16", cuda) for m in (n * k, n))

    def step(stream=None):
        rows, order = pkg.dispatch_sorted(x, ids, E, stream=stream)
        out = pkg.combine_sorted(y, order, w, stream=stream)
        return [rows, out, *torch.autograd.grad([rows, out], [x, y, w], [d_rows, d_out])]
    want = [t.detach().clone() for t in step()]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = step(s)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    got = step(s.cuda_stream)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    with torch.no_grad():
        x.mul_(2.0)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for st, (g, _) in zip((a, b), graphs):
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    want = [t.detach() for t in step()]
    for _, outs in graphs:
        assert all(torch.equal(p, q) for p, q in zip(want, outs))
    assert pkg.moe_cache.device_error() == 0


def test_equal_calls_give_equal_bits(pkg, cuda):
    rng = np.random.default_rng(9)
    n, k, E, H = 3000, 8, 64, 256
    ids = torch.from_numpy(draw_ids(rng, n, k, E)).to(cuda)
    y = rand(rng, (n * k, H), "bf16", cuda).requires_grad_()
    w = torch.rand((n, k), device=cuda).requires_grad_()
    d = rand(rng, (n, H), "bf16", cuda)
    runs = []
    for _ in range(3):
        order = pkg.sort_by_expert(ids, E)
        out = pkg.combine_sorted(y, order, w)
        runs.append([order.rows, out, *torch.autograd.grad(out, [y, w], d)])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], r))


def test_rows_past_32_bits(pkg, cuda):
    """n_tok k H above 2^32 elements: 1200 x 4 rows of 2^20 values."""
    n, k, E, H = 1200, 4, 3, 1 << 20
    g = torch.Generator(device=cuda).manual_seed(1)
    ids = torch.randint(0, E, (n, k), generator=g, device=cuda, dtype=torch.int32)
    x = torch.randn((n, H), generator=g, device=cuda).to(torch.bfloat16)
    rows, order = pkg.dispatch_sorted(x, ids, E)
    at = order.rows.long()
    for p in (0, 2500, n * k - 1):
        assert torch.equal(rows[p], x[at[p] // k])
    w = torch.zeros((n, k), device=cuda)
    w[:, 1] = 1.0
    out = pkg.combine_sorted(rows, order, w)
    assert torch.equal(out[n - 1], x[n - 1]) and torch.equal(out[0], x[0]) and torch.equal(out[700], x[700])
    wl, rl = w.requires_grad_(), rows.requires_grad_()
    d_y, = torch.autograd.grad(pkg.combine_sorted(rl, order, wl), [rl], x)
    assert torch.equal(d_y[order.positions[n - 1, 1]], x[n - 1])
    assert not d_y[order.positions[n - 1, 0]].any()


def test_no_tokens(pkg, cuda):
    ids = torch.empty((0, 4), dtype=torch.int32, device=cuda)
    x = torch.empty((0, 32), device=cuda, requires_grad=True)
    rows, order = pkg.dispatch_sorted(x, ids, 8)
    assert rows.shape == (0, 32) and not order.offsets.any()
    out = pkg.combine_sorted(rows, order, torch.empty((0, 4), device=cuda))
    assert out.shape == (0, 32)
    assert torch.autograd.grad(out.sum(), x)[0].shape == (0, 32)


def test_capture_next_to_an_eager_graph_of_the_same_leaves(pkg, cuda):
    """Autograd would make the capture wait for the eager graph's stream: refused, and fine once that graph is gone or
    where it was made on the capture's stream."""
    rng = np.random.default_rng(10)
    n, k, E, H = 20, 3, 5, 64
    ids = torch.from_numpy(draw_ids(rng, n, k, E)).to(cuda)
    x, y = (rand(rng, (m, H), "f32", cuda).requires_grad_() for m in (n, n * k))
    w = torch.rand((n, k), device=cuda).requires_grad_()
    d = rand(rng, (n, H), "f32", cuda)

    def step(stream):
        with torch.cuda.stream(stream):
            rows, order = pkg.dispatch_sorted(x, ids, E)
            out = pkg.combine_sorted(y, order, w)
            return (rows, out), torch.autograd.grad(out, [y, w], d, retain_graph=True)
    main, side = torch.cuda.current_stream(), torch.cuda.Stream()
    alive, want = step(main)
    want = [t.clone() for t in want]
    torch.cuda.synchronize()
    order = pkg.sort_by_expert(ids, E)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        for call in (lambda: pkg.dispatch_sorted(x, ids, E), lambda: pkg.gather_sorted(x, order), lambda: pkg.combine_sorted(y, order, w)):
            with pytest.raises(pkg.MoeError, match="alive"):
                call()
        with torch.no_grad():
            pkg.combine_sorted(y, order, w)
    del alive
    kept, _ = step(side)                          # (on the capture's stream)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        outs, grads = step(side)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, grads))
    del kept, outs


def test_dispatch_is_sort_and_gather(pkg, cuda):
    """Both forms, about the size where they change."""
    rng = np.random.default_rng(11)
    for n, k, E in ((1, 8, 1024), (255, 8, 64), (256, 8, 300), (257, 8, 64), (682, 3, 1000), (2048, 1, 7), (2049, 1, 7)):
        ids = draw_ids(rng, n, k, E, 0.1)
        if n > 200:
            ids[5, 0] = E
        t = torch.from_numpy(ids).to(cuda)
        x = rand(rng, (n, 72), "bf16", cuda)
        rows, order = pkg.dispatch_sorted(x, t, E)
        check_order(order, ids, E)
        assert pkg.moe_cache.device_error() == (pkg.moe_cache.DERR_BAD_ID if n > 200 else 0)
        other = pkg.sort_by_expert(t, E)
        assert torch.equal(other._buf, order._buf) and torch.equal(rows, pkg.gather_sorted(x, other))
        assert pkg.moe_cache.device_error() == (pkg.moe_cache.DERR_BAD_ID if n > 200 else 0)


def test_results_may_be_written_in_place(pkg, cuda):
    rng = np.random.default_rng(12)
    n, k, E, H = 30, 2, 4, 16
    ids = torch.from_numpy(draw_ids(rng, n, k, E)).to(cuda)
    x = rand(rng, (n, H), "f32", cuda).requires_grad_()
    w = torch.rand((n, k), device=cuda)
    rows, order = pkg.dispatch_sorted(x, ids, E)
    rows.mul_(2.0)
    other = pkg.gather_sorted(x, order).mul_(2.0)
    assert torch.equal(rows, other)
    out = pkg.combine_sorted(rows, order, w).add_(1.0)
    g, = torch.autograd.grad(out, x, torch.ones_like(out))
    want = 2.0 * w.sum(1, keepdim=True).expand(n, H)
    assert (g - want).abs().max() <= 1e-6 * want.abs().max()       # sums of two products: 3 roundings of 2^-24
    rows, order = pkg.dispatch_sorted(x, ids, E)
    out = pkg.combine_sorted(rows, order, w.requires_grad_())
    with torch.no_grad():
        rows.add_(1.0)                                              # saved for d_weights
    with pytest.raises(RuntimeError, match="modified"):
        out.sum().backward()


def test_calls_at_once_on_two_streams(pkg, cuda):
    rng = np.random.default_rng(13)
    jobs = []
    for n, k, E, H in ((5000, 4, 40, 96), (700, 3, 16, 33)):
        ids = torch.from_numpy(draw_ids(rng, n, k, E, 0.1)).to(cuda)
        x, w = rand(rng, (n, H), "bf16", cuda), torch.rand((n, k), device=cuda)
        rows, order = pkg.dispatch_sorted(x, ids, E)
        jobs.append((ids, E, x, w, rows, order._buf.clone(), pkg.combine_sorted(rows, order, w), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(8):
        got = []
        for ids, E, x, w, *_, st in jobs:
            with torch.cuda.stream(st):
                rows, order = pkg.dispatch_sorted(x, ids, E)
                got.append((rows, order._buf, pkg.combine_sorted(rows, order, w)))
        torch.cuda.synchronize()
        for job, g in zip(jobs, got):
            assert all(torch.equal(a, b) for a, b in zip(job[4:7], g))


def test_refusals(pkg, cuda):
    ids = torch.zeros((4, 2), dtype=torch.int32, device=cuda)
    x, y, w = torch.zeros((4, 8), device=cuda), torch.zeros((8, 8), device=cuda), torch.zeros((4, 2), device=cuda)
    order = pkg.sort_by_expert(ids, 3)
    for f in (lambda: pkg.sort_by_expert(ids.long(), 3), lambda: pkg.sort_by_expert(ids[:, 0], 3), lambda: pkg.sort_by_expert(ids.t(), 3),
              lambda: pkg.sort_by_expert(ids[:1].expand(4, 2), 3), lambda: pkg.sort_by_expert(ids, 0), lambda: pkg.sort_by_expert(ids, 1025),
              lambda: pkg.gather_sorted(x[:3], order), lambda: pkg.gather_sorted(x.double(), order), lambda: pkg.gather_sorted(x.t(), order),
              lambda: pkg.gather_sorted(x.cpu(), order), lambda: pkg.gather_sorted(x[:, :0], order), lambda: pkg.gather_sorted(x[0], order),
              lambda: pkg.gather_sorted(x[:1].expand(4, 8), order), lambda: pkg.dispatch_sorted(x[:3], ids, 3),
              lambda: pkg.combine_sorted(x, order, w), lambda: pkg.combine_sorted(y, order, w.half()), lambda: pkg.combine_sorted(y, order, w[:3]),
              lambda: pkg.combine_sorted(y, order, w.t().contiguous().t()), lambda: pkg.combine_sorted(y, order, None),
              lambda: pkg.combine_sorted(y, order, w, shared=x.half()), lambda: pkg.combine_sorted(y, order, w, shared=x[:, :4]),
              lambda: pkg.combine_sorted(y, order, w, shared=x[:3])):
        with pytest.raises(pkg.MoeError):
            f()
    assert pkg.moe_cache.device_error() == 0


def test_uses_between_the_forms(pkg, cuda):
    """Rows long enough that few entries would fill the GPU several times with CTAs that all sort."""
    rng = np.random.default_rng(14)
    for n, k, E, H in ((2000, 1, 30, 2048), (300, 2, 9, 9000)):
        ids = draw_ids(rng, n, k, E, 0.1)
        x = rand(rng, (n, H), "bf16", cuda)
        rows, order = pkg.dispatch_sorted(x, torch.from_numpy(ids).to(cuda), E)
        ref_rows = check_order(order, ids, E)[0]
        live = torch.from_numpy(ref_rows[ref_rows >= 0]).to(cuda).long()
        assert torch.equal(rows[: live.numel()], x[live // k]) and not rows[live.numel():].any()


@pytest.mark.parametrize("n", [4095, 4096, 9001])      # 8 picks each: below, at and above the larger cluster's first size
def test_many_entries_of_a_wider_buffer_in_a_graph(pkg, cuda, n):
    rng = np.random.default_rng(n)
    E, k, H = 100, 8, 24
    wide = draw_ids(rng, n, 11, E, 0.1)
    wide[n // 2, 3], wide[n - 1, 8] = E, -7           # as empty slots, and reported
    t, x = torch.from_numpy(wide).to(cuda), rand(rng, (n, H), "bf16", cuda)
    pkg.dispatch_sorted(x, t[:, 2:10], E)
    assert pkg.moe_cache.device_error() == pkg.moe_cache.DERR_BAD_ID
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rows, order = pkg.dispatch_sorted(x, t[:, 2:10], E)
        alone = pkg.sort_by_expert(t[:, 2:10], E)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    r, _, _, offsets = check_order(order, wide[:, 2:10], E)
    check_order(alone, wide[:, 2:10], E)
    live = offsets[-1]
    assert torch.equal(rows[:live], x[torch.from_numpy(r[:live] // k).long().to(cuda)]) and not rows[live:].any()
    assert pkg.moe_cache.device_error() == pkg.moe_cache.DERR_BAD_ID and pkg.moe_cache.device_error() == 0
