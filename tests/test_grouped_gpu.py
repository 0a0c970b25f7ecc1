"""Products grouped by expert on the GPU against 64-bit products, group by group.

Tolerance of a result: its final rounding (half a step of its type, relative) and the fp32 sum. The tensor core adds
sixteen products at a time into a 24-bit sum, and an add is off by at most 2^-23 of the partial sums' size (it may truncate), which
the sum of the magnitudes bounds: (ceil(K / 16) + 16) * 2^-23 * sum |a||b|."""
import numpy as np
import pytest

import t2sp_b200
from t2sp_b200 import GroupedDesc
from tests.device_util import buf, eps_half, on_stream

pytestmark = pytest.mark.gpu


def make(E, K, N, counts, dtype, trans=False, before=0, behind=0, seed=0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    M = before + sum(counts) + behind
    a = torch.randn(M, K, generator=g, device="cuda").to(dtype)
    b = torch.randn(E, *((N, K) if trans else (K, N)), generator=g, device="cuda").to(dtype)
    d = torch.randn(M, N, generator=g, device="cuda").to(dtype)
    off = torch.tensor(np.concatenate([[before], before + np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    return a, b, d, off


def close(got, ref, mag, terms):
    """|got - ref| within the tolerance above, element by element."""
    import torch
    tol = eps_half(got.dtype) * ref.abs() if got.dtype != torch.float32 else 0
    tol = tol + ((terms + 15) // 16 + 16) * 2.0 ** -23 * mag * (1 + eps_half(got.dtype)) + 1e-30
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25     # below fp16's smallest normal number a step is 2^-24
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got.double() - ref).abs().max()))


def check_forward(a, b, off, c, trans, untouched):
    import torch
    o = off.tolist()
    for e in range(len(o) - 1):
        lo, hi = o[e], o[e + 1]
        if hi > lo:
            w = (b[e].T if trans else b[e]).double()
            close(c[lo:hi], a[lo:hi].double() @ w, a[lo:hi].double().abs() @ w.abs(), a.shape[1])
    assert torch.equal(c[:o[0]], untouched[:o[0]]) and torch.equal(c[o[-1]:], untouched[o[-1]:])


def check_grad(a, d, off, g):
    o = off.tolist()
    for e in range(len(o) - 1):
        x, y = a[o[e]:o[e + 1]].double(), d[o[e]:o[e + 1]].double()
        if o[e + 1] == o[e]:
            assert not g[e].any() and not g[e].isnan().any()
        else:
            close(g[e], x.T @ y, x.abs().T @ y.abs(), o[e + 1] - o[e])


SHAPES = [
    # counts, K, N, rows before, rows behind
    ([1], 64, 64, 0, 0),
    ([1, 0, 2, 0], 16, 8, 0, 0),
    ([0, 0], 128, 128, 0, 5),
    ([5, 64, 1, 31, 33, 0, 127], 136, 264, 0, 0),
    ([256, 257, 255, 1], 512, 256, 0, 3),
    ([300, 0, 41], 1000, 520, 7, 9),
    ([3, 2, 0, 6], 37, 45, 0, 1),
    ([70, 90], 65, 33, 2, 0),
    ([40, 9], 1, 1, 0, 0),
    ([600, 20], 72, 1032, 0, 0),
    ([1] * 300, 64, 128, 0, 0),
    ([20, 200], 2056, 24, 0, 0),
    ([0, 1700, 0, 0, 900], 256, 776, 0, 16),
    ([129, 71] * 8, 1024, 100, 0, 3),      # uneven groups: more tiles than an even spread would give
    ([3], 4104, 136, 1, 1),
    ([2, 1], 320, 1000, 0, 0),
    ([2100, 300], 2112, 1032, 0, 0),
    ([64, 5, 0, 300], 1379, 1188, 0, 2),   # rows that do not start on 16 bytes, many blocks and tiles
    ([20] * 12, 1222, 1417, 0, 0),
    ([7], 5378, 187, 0, 1),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d_%d" % (s[1], s[2], sum(s[0])))
def test_forward(lib, shape, trans, dtype):
    import torch
    counts, K, N, before, behind = shape
    dt = getattr(torch, dtype)
    a, b, _, off = make(len(counts), K, N, counts, dt, trans, before, behind)
    for out in (dt, torch.float32):
        c = torch.full((a.shape[0], N), 7.0, dtype=out, device="cuda")
        with on_stream():
            assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c), GroupedDesc(int(trans))) == 0
        check_forward(a, b, off, c, trans, torch.full_like(c, 7.0))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d_%d" % (s[1], s[2], sum(s[0])))
def test_grad(lib, shape, dtype):
    import torch
    counts, K, N, before, behind = shape
    dt = getattr(torch, dtype)
    a, _, d, off = make(len(counts), K, N, counts, dt, False, before, behind)
    for out in (dt, torch.float32):
        g = torch.full((len(counts), K, N), float("nan"), dtype=out, device="cuda")
        with on_stream():
            assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
        check_grad(a, d, off, g)


def test_rows_of_others_do_not_leak(lib):
    """Rows outside the groups, and the rows of a neighbouring group, hold NaN and infinities."""
    import torch
    counts, K, N = [30, 45, 21], 200, 136
    a, b, d, off = make(3, K, N, counts, torch.bfloat16, before=3, behind=40)
    o = off.tolist()
    a[:o[0]] = float("nan"); a[o[1]:o[2]] = float("inf"); a[o[3]:] = float("nan")
    d[:o[0]] = float("inf"); d[o[1]:o[2]] = float("nan"); d[o[3]:] = float("nan")
    c = torch.full((a.shape[0], N), 7.0, dtype=torch.bfloat16, device="cuda")
    g = torch.empty(3, K, N, dtype=torch.bfloat16, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c)) == 0
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
    for e in (0, 2):
        lo, hi = o[e], o[e + 1]
        close(c[lo:hi], a[lo:hi].double() @ b[e].double(), a[lo:hi].double().abs() @ b[e].double().abs(), K)
        x, y = a[lo:hi].double(), d[lo:hi].double()
        close(g[e], x.T @ y, x.abs().T @ y.abs(), hi - lo)
    assert not c[o[1]:o[2]].isfinite().any() and g[1].isnan().all()
    assert (c[:o[0]] == 7).all() and (c[o[3]:] == 7).all()


@pytest.mark.parametrize("pad_a,pad_b,pad_c,first", [(8, 8, 8, 0), (3, 0, 1, 0), (0, 5, 0, 1), (8, 16, 3, 1)])
def test_strides_and_offsets_of_operands(lib, pad_a, pad_b, pad_c, first):
    """Padded rows and matrices, and operands that start inside an allocation (first = 1: not on 16 bytes)."""
    import torch
    counts, K, N = [33, 0, 50], 120, 72
    a0, b0, d0, off = make(3, K, N, counts, torch.float16)
    M = sum(counts)

    def inside(t, pad):
        big = torch.full((t.numel() // t.shape[-1] * (t.shape[-1] + pad) + 64,), float("nan"), dtype=t.dtype, device="cuda")
        view = big[first:].as_strided(t.shape, [s // t.shape[-1] * (t.shape[-1] + pad) if i < t.dim() - 1 else 1 for i, s in enumerate(t.stride())])
        view.copy_(t)
        return big, view
    _, a = inside(a0, pad_a)
    _, b = inside(b0, pad_b)
    _, d = inside(d0, pad_b)
    cbig, c = inside(torch.zeros(M, N, dtype=torch.float16, device="cuda"), pad_c)
    gbig, g = inside(torch.zeros(3, K, N, dtype=torch.float16, device="cuda"), pad_c)
    holes = cbig.isnan().sum().item(), gbig.isnan().sum().item()
    with on_stream():
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c)) == 0
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
    check_forward(a0, b0, off, c, False, c)
    check_grad(a0, d0, off, g)
    assert holes == (cbig.isnan().sum().item(), gbig.isnan().sum().item())   # nothing was written between the rows


def test_matrices_interleaved_by_rows(lib):
    """B(n, k, e) with e between n and k in memory."""
    import torch
    a, b0, d, off = make(3, 64, 80, [10, 20, 30], torch.bfloat16)
    b = torch.empty(64, 3, 80, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    b.copy_(b0)
    g = torch.empty(64, 3, 80, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    c = torch.empty(60, 80, dtype=torch.bfloat16, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c)) == 0
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
    check_forward(a, b0, off, c, False, c)
    check_grad(a, d, off, g)


@pytest.mark.parametrize("offsets", [[0, 10, 5, 20], [-1, 3, 5, 20], [0, 3, 5, 21], [0, 2 ** 31 - 1, 5, 20]])
def test_bad_offsets_compute_nothing(lib, offsets):
    import torch
    a, b, d, _ = make(3, 64, 64, [10, 5, 5], torch.bfloat16)
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    c = torch.full((20, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    g = torch.full((3, 64, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c)) == -4
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == -4
    assert (c == 7).all() and (g == 7).all()
    with on_stream(asynchronous=True) as L:
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c)) == 0
        assert L.t2sp_b200_sync() == -4 and L.t2sp_b200_sync() == 0    # reported once


def test_empty_contractions_and_no_rows(lib):
    import torch
    off = torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    c = torch.full((6, 8), 7.0, dtype=torch.bfloat16, device="cuda")
    a, b = torch.empty(6, 0, dtype=torch.bfloat16, device="cuda"), torch.empty(2, 0, 8, dtype=torch.bfloat16, device="cuda")
    A = t2sp_b200.Buffer((0, 6), "bf16", host=c.data_ptr())       # nothing of an empty operand is read
    B = t2sp_b200.Buffer((8, 0, 2), "bf16", host=c.data_ptr())
    with on_stream():
        assert t2sp_b200.grouped_gemm(A, B, buf(off), buf(c)) == 0
        assert not c[:5].any() and (c[5:] == 7).all()
        none = torch.zeros(3, dtype=torch.int32, device="cuda")
        g = torch.full((2, 8, 16), 7.0, dtype=torch.float32, device="cuda")
        X = t2sp_b200.Buffer((8, 0), "bf16", host=c.data_ptr())
        Y = t2sp_b200.Buffer((16, 0), "bf16", host=c.data_ptr())
        assert t2sp_b200.grouped_gemm_grad(X, Y, buf(none), buf(g)) == 0
        assert not g.any()


def test_host_buffers(lib):
    """Host operands travel like those of the other operators; rows outside the groups come back as they were."""
    import torch
    from t2sp_b200 import Buffer
    a, b, d, off = make(3, 40, 56, [4, 0, 7], torch.bfloat16, before=2, behind=3)

    def host(t):
        return Buffer.from_numpy(t.cpu().view(torch.int16).numpy().view(np.uint16), dtype="bf16")
    c = np.full((a.shape[0], 56), 3.0, np.float32)
    C = Buffer.from_numpy(c)
    assert t2sp_b200.grouped_gemm(host(a), host(b), Buffer.from_numpy(off.cpu().numpy()), C) == 0
    got = torch.from_numpy(C.keepalive).cuda()
    check_forward(a, b, off, got, False, torch.full_like(got, 3.0))
    G = Buffer.from_numpy(np.zeros((3, 40, 56), np.float32))
    assert t2sp_b200.grouped_gemm_grad(host(a), host(d), Buffer.from_numpy(off.cpu().numpy()), G) == 0
    check_grad(a, d, off, torch.from_numpy(G.keepalive).cuda())


def test_gradients_against_differences(lib):
    """f = sum(D * forward(A, B)) is linear in A and in B: f(x + v) - f(x - v) = 2 <gradient, v>, up to the fp32 results' errors."""
    import torch
    counts, K, N = [17, 0, 40], 96, 64
    a, b, d, off = make(3, K, N, counts, torch.bfloat16)
    M = sum(counts)
    da = torch.empty(M, K, dtype=torch.float32, device="cuda")
    db = torch.empty(3, K, N, dtype=torch.float32, device="cuda")

    def f(a, b):   # the value, and a bound of its error from the fp32 sums (see the module's tolerance)
        c = torch.empty(M, N, dtype=torch.float32, device="cuda")
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c)) == 0
        o = off.tolist()
        mag = torch.cat([a[o[e]:o[e + 1]].double().abs() @ b[e].double().abs() for e in range(3)])
        return float((c.double() * d.double()).sum()), (K / 16 + 16) * 2.0 ** -23 * float((mag * d.abs().double()).sum())
    with on_stream():
        assert t2sp_b200.grouped_gemm(buf(d), buf(b), buf(off), buf(da), GroupedDesc(1)) == 0
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(db)) == 0
        for x, g, at in ((a, da, lambda y: f(y, b)), (b, db, lambda y: f(a, y))):
            v = torch.zeros_like(x)
            v.view(-1)[::7] = 1.0
            lo, hi = x - v, x + v
            step = hi.double() - lo.double()       # what the roundings to bf16 left of 2 v
            (f1, t1), (f0, t0) = at(hi), at(lo)
            # the gradient's own error is bounded the same way: |step| takes the place of the moved operand
            o = off.tolist()
            if x is a:
                mag = torch.cat([step[o[e]:o[e + 1]].abs() @ b[e].double().abs() for e in range(3)])
            else:
                mag = torch.cat([a[o[e]:o[e + 1]].double().abs() @ step[e].abs() for e in range(3)])
            tol = t1 + t0 + (max(N, max(counts)) / 16 + 16) * 2.0 ** -23 * float((mag * d.abs().double()).sum())
            want = float((g.double() * step).sum())
            assert abs((f1 - f0) - want) <= tol, (f1 - f0, want, tol)


def test_graph_and_streams(lib):
    """Forward and backward captured once and replayed with other rows and other group boundaries; eager calls on a second stream meanwhile."""
    import torch
    K, N, E = 128, 192, 4
    a, b, d, off = make(E, K, N, [50, 0, 70, 30], torch.bfloat16)
    c = torch.zeros(150, N, dtype=torch.bfloat16, device="cuda")
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    side = torch.cuda.Stream()

    def step():
        assert t2sp_b200.grouped_gemm(A, B, O, C) == 0
        assert t2sp_b200.grouped_gemm(D, B, O, DA, GroupedDesc(1)) == 0
        assert t2sp_b200.grouped_gemm_grad(A, D, O, DB) == 0
    A, B, C, D, O, DA, DB = (buf(t) for t in (a, b, c, d, off, da, db))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with on_stream(side, asynchronous=True):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            step()
    for counts, seed in (([150, 0, 0, 0], 1), ([1, 2, 3, 140], 2)):
        a2, b2, d2, off2 = make(E, K, N, counts, torch.bfloat16, behind=150 - sum(counts), seed=seed)
        for t, u in ((a, a2), (b, b2), (d, d2), (off, off2)):
            t.copy_(u)
        c.fill_(5); da.fill_(5)
        torch.cuda.synchronize()
        graph.replay()
        other = torch.cuda.Stream()
        x, w, y, o = make(2, 64, 64, [100, 31], torch.bfloat16, seed=9)
        z = torch.zeros(131, 64, dtype=torch.bfloat16, device="cuda")
        torch.cuda.current_stream().synchronize()
        with on_stream(other):
            assert t2sp_b200.grouped_gemm(buf(x), buf(w), buf(o), buf(z)) == 0
        torch.cuda.synchronize()
        check_forward(a, b, off, c, False, torch.full_like(c, 5))
        check_forward(d, b, off, da, True, torch.full_like(da, 5))
        check_grad(a, d, off, db)
        check_forward(x, w, o, z, False, z)


def test_capture_refuses_what_it_cannot_hold(lib):
    """A synchronous call, and a call that needs scratch memory, are refused inside a capture, which goes on."""
    import torch
    a, b, _, off = make(2, 37, 64, [10, 20], torch.bfloat16)
    good, wide, _, _ = make(2, 64, 64, [10, 20], torch.bfloat16)
    c = torch.zeros(30, 64, dtype=torch.bfloat16, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    bufs = [buf(t) for t in (a, b, off, c, good, wide)]
    torch.cuda.synchronize()
    with on_stream(side, asynchronous=True) as L:
        assert t2sp_b200.grouped_gemm(bufs[4], bufs[5], bufs[2], bufs[3]) == 0
        side.synchronize()
        c.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            rc_scratch = t2sp_b200.grouped_gemm(bufs[0], bufs[1], bufs[2], bufs[3])
            L.t2sp_b200_set_async(0)
            rc_sync = t2sp_b200.grouped_gemm(bufs[4], bufs[5], bufs[2], bufs[3])
            L.t2sp_b200_set_async(1)
            rc_ok = t2sp_b200.grouped_gemm(bufs[4], bufs[5], bufs[2], bufs[3])
    assert (rc_scratch, rc_sync, rc_ok) == (-8, -8, 0)
    graph.replay()
    torch.cuda.synchronize()
    check_forward(good, wide, off, c, False, c)


def test_repeatable(lib):
    import torch
    a, b, d, off = make(5, 520, 776, [100, 3, 0, 900, 77], torch.bfloat16)
    outs = []
    for _ in range(2):
        c = torch.zeros(a.shape[0], 776, dtype=torch.float32, device="cuda")
        g = torch.zeros(5, 520, 776, dtype=torch.float32, device="cuda")
        with on_stream():
            assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c)) == 0
            assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
        outs.append((c, g))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_long_fp32_gradient(lib):
    """An fp32 gradient over many rows is added up in runs of 512. With values of random sign (deviation s for a product) a run's
    partial sums have about 12 s on the mean; 32 steps that cut off 2^-24 of them on the mean give 2.3e-5 s a run, over 79 runs in
    quadrature 2e-4 s, of a result of 200 s: 1e-6 relative in the 2-norm, 5e-6 with room. One sum over all rows would be 5e-5 off."""
    import torch
    a, _, d, off = make(1, 256, 256, [40000], torch.bfloat16)
    g = torch.empty(1, 256, 256, dtype=torch.float32, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
    ref = a.double().T @ d.double()
    assert float((g[0].double() - ref).norm() / ref.norm()) <= 5e-6


def test_two_threads_on_their_own_streams(lib):
    """Two host threads call at once, each on its own stream, one of them with operands that need scratch memory."""
    import threading

    import torch
    made = [make(3, 64 + 5 * i, 128, [100, 0, 57], torch.bfloat16, seed=i) for i in range(2)]
    outs = [torch.zeros(157, 128, dtype=torch.bfloat16, device="cuda") for _ in made]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            a, b, _, off = made[i]
            stream = torch.cuda.Stream()
            with on_stream(stream, asynchronous=True) as L:
                for _ in range(50):
                    assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(outs[i])) == 0
                assert L.t2sp_b200_sync() == 0
        except BaseException as e:   # reported by the main thread
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for (a, b, _, off), c in zip(made, outs):
        check_forward(a, b, off, c, False, c)


@pytest.mark.parametrize("trans", [False, True])
def test_more_tiles_than_are_listed(lib, trans):
    """A worker's tiles beyond the ones it prepares at the start, with a narrow last block of columns: 900 groups of a row, 9 blocks of n."""
    import torch
    E, K, N = 900, 8, 2056
    a, b, _, off = make(E, K, N, [1] * E, torch.bfloat16, trans, 2, 3)
    c = torch.full((a.shape[0], N), 7.0, dtype=torch.bfloat16, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c), GroupedDesc(int(trans))) == 0
    x, w = a[2:2 + E].double().unsqueeze(1), (b.transpose(1, 2) if trans else b).double()
    close(c[2:2 + E], torch.bmm(x, w).squeeze(1), torch.bmm(x.abs(), w.abs()).squeeze(1), K)
    assert (c[:2] == 7).all() and (c[2 + E:] == 7).all()


@pytest.mark.parametrize("E", [128, 1000])
def test_grad_of_many_tiles(lib, E):
    """The same for the gradient: long and short groups in the order of their rows (up to 128 groups) or as they come, narrow last blocks of n and of k."""
    import torch
    K, N = (520, 4104) if E == 128 else (8, 2056)
    counts = [3 + 11 * (e % 5) for e in range(E)]
    counts[17], counts[90], counts[91] = 700, 0, 333
    a, _, d, off = make(E, K, N, counts, torch.bfloat16, False, 1, 2)
    g = torch.full((E, K, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
    check_grad(a, d, off, g)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,counts,K,N,skip", [
    ("split", [7], 4096, 128, 3), ("split", [100], 4096, 128, 2), ("single", [600, 400], 512, 512, 3), ("pair", [4000, 96], 512, 1024, 3),
    ("warps", [10] * 20, 515, 1031, 3), ("grad", [700], 512, 256, 3), ("grad", [40], 512, 256, 1)])
def test_bounded_waits_run_out(lib, name, counts, K, N, skip, out):
    """Without the copies from one k-block on (a test hook) the waits behind it run out after the shortened limit: every kernel returns by
    itself, in each of its tile variants, the call reports it, and the next call is right."""
    import torch
    from tests.util import library_env
    a, b, d, off = make(len(counts), K, N, counts, torch.bfloat16)
    dt = getattr(torch, out)
    c = torch.zeros(a.shape[0], N, dtype=dt, device="cuda")
    g = torch.zeros(len(counts), K, N, dtype=dt, device="cuda")

    def call():
        with on_stream():
            if name == "grad":
                return t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g))
            return t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c))
    with library_env(T2SP_B200_WAIT_CYCLES="20000000", T2SP_B200_TEST_SKIP_STAGE=str(skip)):
        assert call() == -23
    assert call() == 0
    if name == "grad":
        check_grad(a, d, off, g)
    else:
        check_forward(a, b, off, c, False, c)


@pytest.mark.parametrize("name", ["grouped_gemm", "grouped_gemm_grad", "q4_gemv"])
def test_newer_host_values_of_a_resident_output_stay(lib, name):
    """An output with a device allocation whose host side was changed (host_dirty): what the call does not write comes back from
    copy_to_host as the host had it."""
    import torch
    from t2sp_b200 import Buffer, Q4Desc
    from tests.device_util import packed
    a, b, d, off = make(2, 64, 48, [5, 4], torch.bfloat16, before=2, behind=3)
    w = b.contiguous()
    M, K, N = a.shape[0], 64, 48
    shape = {"grouped_gemm": (M, N + 8), "grouped_gemm_grad": (2, K + 2, N + 8), "q4_gemv": (M, N)}[name]
    out = np.zeros(shape, np.float32)
    C = Buffer.from_numpy(out)
    assert lib.t2sp_b200_device_malloc(C.ptr) == 0 and lib.t2sp_b200_copy_to_device(C.ptr) == 0
    out[:] = 7.0
    C.raw.flags |= 1   # host_dirty
    with on_stream():
        if name == "grouped_gemm":
            rc = t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), C)
        elif name == "grouped_gemm_grad":
            rc = t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), C)
        else:
            Q, S = packed(w, 64)
            index = torch.tensor([-1, 0, 1, -1] + [0] * (M - 4), dtype=torch.int32, device="cuda")
            rc = t2sp_b200.q4_gemv(buf(a), buf(Q), buf(S), buf(index), C, Q4Desc(64, 0))
    assert rc == 0 and not C.raw.flags & 1
    assert lib.t2sp_b200_copy_to_host(C.ptr) == 0 and lib.t2sp_b200_device_free(C.ptr) == 0
    got = torch.from_numpy(out).cuda()
    if name == "grouped_gemm":
        check_forward(a, b, off, got[:, :N], False, torch.full_like(got, 7.0)[:, :N])
        assert (got[:, N:] == 7).all()
    elif name == "grouped_gemm_grad":
        check_grad(a, d, off, got[:, :K, :N])
        assert (got[:, K:] == 7).all() and (got[:, :, N:] == 7).all()
    else:
        assert (got[[0, 3]] == 7).all() and not (got[[1, 2, 4]] == 7).any()


def long_tolerance(ref):
    """All products positive. Beside the final rounding to f16 (2^-11): runs of 512 steps, each of which cuts off less than 2^-23 of the sum
    (2^-14), and fewer than 512 sums of runs or parts in fp32 (2^-15), relative. One sum over 2^17 rows would be 8e-4 low, over 2^20 7e-3."""
    return ref * (2.0 ** -11 + 2.0 ** -14 + 2.0 ** -15) * (1 + 2.0 ** -11)


def positive(seed, *shape):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.rand(*shape, generator=g, device="cuda") * 0.1 + 0.1).half()


def test_long_f16_gradient(lib):
    """A group of 2^20 rows, an empty one, one of 40 rows and one of 2^17."""
    import torch
    counts = [(1 << 20) + 37, 0, 40, 1 << 17]
    rows = sum(counts)
    a, d = positive(3, rows, 72), positive(4, rows, 88)
    off = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    out = torch.empty(4, 72, 88, dtype=torch.float16, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(out)) == 0
    o = off.tolist()
    for e in (0, 2, 3):
        ref = sum(a[i:min(o[e + 1], i + 65536)].double().T @ d[i:min(o[e + 1], i + 65536)].double() for i in range(o[e], o[e + 1], 65536))
        assert ((out[e].double() - ref).abs() <= long_tolerance(ref)).all(), e
    assert not out[1].any()


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("counts,K,N", [([5, 0, 30], 140000, 40), ([3, 300], 131085, 300), ([20], 60000, 136), ([2000, 3000], 131072, 1032)])
def test_long_f16_contractions(lib, counts, K, N, trans):
    """Few tiles (with the contraction shared by a cluster up to 65536 k), and many."""
    import torch
    E, M = len(counts), sum(counts) + 3
    a, b = positive(5, M, K), positive(6, E, *((N, K) if trans else (K, N)))
    off = torch.tensor(1 + np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    c = torch.full((M, N), 7.0, dtype=torch.float16, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c), GroupedDesc(int(trans))) == 0
    o = off.tolist()
    for e in range(E):
        if counts[e]:
            w = b[e].T if trans else b[e]
            ref = sum(a[o[e]:o[e + 1], k:k + 16384].double() @ w[k:k + 16384].double() for k in range(0, K, 16384))
            assert ((c[o[e]:o[e + 1]].double() - ref).abs() <= long_tolerance(ref)).all(), e
    assert (c[:1] == 7).all() and (c[o[-1]:] == 7).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("counts,K,N", [([5, 0, 30], 8200, 1040), ([3, 300] * 20, 8193, 300), ([700, 900], 16500, 1100)])
def test_contractions_of_some_runs(lib, counts, K, N, trans, dtype):
    import torch
    dt = getattr(torch, dtype)
    a, b, d, off = make(len(counts), K, N, counts, dt, trans, 1, 2)
    a, b = a * 2.0 ** -6, b * 2.0 ** -6
    for out in (dt, torch.float32):
        c = torch.full((a.shape[0], N), 7.0, dtype=out, device="cuda")
        with on_stream():
            assert t2sp_b200.grouped_gemm(buf(a), buf(b), buf(off), buf(c), GroupedDesc(int(trans))) == 0
        check_forward(a, b, off, c, trans, torch.full_like(c, 7.0))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_grad_of_long_and_short_groups(lib, dtype):
    """Groups of more and of fewer rows than a run, ragged and empty ones, in one call."""
    import torch
    dt = getattr(torch, dtype)
    counts = [9000, 0, 8192, 8193, 40, 17000, 1, 640] if dtype == "float16" else [70000, 0, 65536, 65537, 40, 140000, 1, 640]
    a, _, d, off = make(len(counts), 200, 264, counts, dt, False, 3, 5)
    g = torch.full((len(counts), 200, 264), float("nan"), dtype=dt, device="cuda")
    with on_stream():
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
    check_grad(a, d, off, g)


def test_matrices_of_an_output_that_interlock(lib):
    """G's rows have a pitch, and a matrix begins where the last row of the one before ends: in device and in host memory."""
    import torch
    from t2sp_b200 import Buffer
    a, _, d, off = make(3, 40, 24, [10, 0, 70], torch.bfloat16)
    big = torch.full((3 * (39 * 32 + 24) + 8,), 5.0, dtype=torch.float32, device="cuda")
    g = big.as_strided((3, 40, 24), (39 * 32 + 24, 32, 1))
    host = big.cpu().numpy().copy()
    with on_stream():
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), buf(g)) == 0
        G = Buffer((24, 40, 3), "f32", host=host.ctypes.data, strides=(1, 32, 39 * 32 + 24), keepalive=host)
        assert t2sp_b200.grouped_gemm_grad(buf(a), buf(d), buf(off), G) == 0
    check_grad(a, d, off, g)
    assert torch.equal(torch.from_numpy(host).cuda(), big)
    g.fill_(5.0)
    assert (big == 5).all()


@pytest.mark.parametrize("trans", [False, True])
def test_long_contraction_off_16_bytes_in_a_capture(lib, trans):
    """B with rows off 16 bytes, read by warps in place: no scratch memory, so the call can be captured, at lengths of several runs too."""
    import torch
    E, K, N = 12, 9005, 1099
    M = 2 * E
    a, b = positive(1, M, K + 3)[:, :K], positive(2, E, *((N, K) if trans else (K, N)))
    a = torch.nn.functional.pad(a, (0, 3))[:, :K]       # rows of A start on 16 bytes
    off = torch.arange(0, M + 1, 2, dtype=torch.int32, device="cuda")
    c = torch.zeros(M, N, dtype=torch.float16, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    A, B, O, C = (buf(t) for t in (a, b, off, c))
    torch.cuda.synchronize()
    with on_stream(side, asynchronous=True):
        assert t2sp_b200.grouped_gemm(A, B, O, C, GroupedDesc(int(trans))) == 0
        side.synchronize()
        c.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            rc = t2sp_b200.grouped_gemm(A, B, O, C, GroupedDesc(int(trans)))
    assert rc == 0
    graph.replay()
    torch.cuda.synchronize()
    for e in range(E):
        ref = a[2 * e:2 * e + 2].double() @ (b[e].T if trans else b[e]).double()
        assert ((c[2 * e:2 * e + 2].double() - ref).abs() <= long_tolerance(ref)).all(), e
