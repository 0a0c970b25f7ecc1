"""4-bit matrices on the GPU: quantising and reading back exactly as the definition in 64 bits says, products with a few rows
against 64-bit products of the values that the integers stand for.

Tolerance of a product: its final rounding (half a step of its type) and the fp32 sums: within a group
(group / 16 + 16) * 2^-23 and over the groups (groups + 16) * 2^-23, of sum |x||w|."""
import numpy as np
import pytest

import t2sp_b200
from t2sp_b200 import Buffer, GroupedDesc, Q4Desc
from tests.device_util import buf, eps_half, on_stream, packed, quantised64

pytestmark = pytest.mark.gpu


def matrices(E, K, N, dtype, seed=0, scale=1.0):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(E, K, N, generator=g, device="cuda") * scale).to(dtype)


def unpacked(Q, S, like, group, trans=False):
    import torch
    w = torch.full_like(like, float("nan"))
    assert t2sp_b200.q4_unpack(buf(Q), buf(S), buf(w), Q4Desc(group, int(trans))) == 0
    return w


def check_rows(x, values, index, y, group, untouched=None):
    """values: (E, K, N) in 64 bits; index: a list, or None."""
    import torch
    R, K = y.shape[0], x.shape[1]
    per = R // x.shape[0]
    index = index if index is not None else [0] * R
    for r in range(R):
        if not 0 <= index[r] < values.shape[0]:
            assert torch.equal(y[r], untouched[r])
            continue
        v, w = x[r // per].double(), values[index[r]]
        ref, mag = v @ w, v.abs() @ w.abs()
        tol = ((group // 16 + 16) + (K // group + 16)) * 2.0 ** -23 * mag + 1e-30
        if y.dtype != torch.float32:
            tol = tol * (1 + eps_half(y.dtype)) + eps_half(y.dtype) * ref.abs() + (2.0 ** -25 if y.dtype == torch.float16 else 0)
        bad = ~((y[r].double() - ref).abs() <= tol)
        assert not bad.any(), (r, int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("E,K,N,group", [(1, 64, 16, 64), (2, 100, 40, 32), (1, 1, 1, 128), (3, 130, 70, 128), (1, 1001, 777, 64),
                                         (2, 256, 128, 32), (1, 192, 33, 128), (5, 63, 17, 32)])
def test_pack_and_unpack_exactly(lib, E, K, N, group, dtype, trans):
    import torch
    dt = getattr(torch, dtype)
    w = matrices(E, K, N, dt, seed=K + N)
    w[:, : K // 3] *= 0.01
    stored = w.transpose(1, 2).contiguous() if trans else w
    with on_stream():
        Q, S = packed(stored, group, trans)
        back = unpacked(Q, S, stored, group, trans)
    want = quantised64(w, group).to(dt)
    assert torch.equal(back.transpose(1, 2) if trans else back, want)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_pack_borders(lib, dtype):
    """Ties, zeros, the smallest and the largest values of the type."""
    import torch
    dt = getattr(torch, dtype)
    fi = torch.finfo(dt)
    w = torch.zeros(1, 64, 48, device="cuda")
    w[0, :, 0] = torch.arange(64) % 15 - 7                     # scale 1: integers and ...
    w[0, :, 1] = (torch.arange(64) % 28 - 14) / 2              # ... halves, ties to even
    w[0, :, 2] = 0
    w[0, 5, 3] = -7
    w[0, :, 4] = fi.max
    w[0, :, 5] = fi.smallest_normal
    w[0, :, 6] = fi.smallest_normal * fi.eps                   # the smallest subnormal number: the scale rounds to zero or not
    w[0, ::2, 7] = fi.smallest_normal * fi.eps * 9
    w[0, :, 8] = -torch.arange(64, device="cuda") * fi.smallest_normal / 8
    w = w.to(dt)
    with on_stream():
        Q, S = packed(w, 64)
        back = unpacked(Q, S, w, 64)
    assert torch.equal(back, quantised64(w, 64).to(dt))


def test_pack_infinities_and_nan(lib):
    """A group with a value that is not finite reads back as nothing finite; the others are as ever."""
    import torch
    w = matrices(1, 128, 40, torch.bfloat16)
    bad = w.clone()
    bad[0, 3, 7] = float("nan"); bad[0, 70, 8] = float("inf"); bad[0, 71, 39] = -float("inf")
    x = torch.ones(1, 128, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(1, 40, dtype=torch.float32, device="cuda")
    with on_stream():
        Q, S = packed(bad, 64)
        back = unpacked(Q, S, bad, 64)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), None, buf(y), Q4Desc(64, 0)) == 0
    want = quantised64(w, 64).to(torch.bfloat16)
    hit = torch.zeros(1, 128, 40, dtype=torch.bool, device="cuda")
    hit[0, :64, 7] = hit[0, 64:, 8] = hit[0, 64:, 39] = True
    assert not back[hit].isfinite().any() and torch.equal(back[~hit], want[~hit])
    columns = hit.any(1)[0]
    assert not y[0][columns].isfinite().any() and y[0][~columns].isfinite().all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,K,N,group", [(1, 64, 16, 64), (1, 1, 1, 32), (1, 4096, 520, 64), (2, 100, 40, 32), (7, 1001, 777, 32), (8, 512, 48, 128),
                                         (9, 130, 33, 128), (17, 192, 64, 64), (33, 256, 80, 32), (70, 64, 17, 64), (3, 8200, 24, 128), (9, 30000, 20, 64),
                                         (1, 65000, 16, 128), (1, 16000, 20, 32), (1100, 64, 16, 64)])
def test_gemv_one_matrix(lib, R, K, N, group, dtype):
    import torch
    dt = getattr(torch, dtype)
    w, x = matrices(1, K, N, dt, 1), matrices(1, R, K, dt, 2)[0]
    with on_stream():
        Q, S = packed(w, group)
        for out in (dt, torch.float32):
            y = torch.full((R, N), float("nan"), dtype=out, device="cuda")
            assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), None, buf(y), Q4Desc(group, 0)) == 0
            check_rows(x, quantised64(w, group), None, y, group)


@pytest.mark.parametrize("E,T,per,K,N,group", [(4, 3, 2, 128, 64, 32), (64, 8, 2, 512, 96, 64), (3, 40, 1, 96, 40, 32), (5, 1, 1, 1000, 24, 128),
                                               (2, 30, 4, 70, 35, 64), (200, 70, 4, 64, 16, 64),
                                               (1, 100, 1, 192, 40, 128), (7, 512, 2, 64, 20, 32)])
def test_gemv_by_expert(lib, E, T, per, K, N, group):
    import torch
    dt = torch.bfloat16
    w, x = matrices(E, K, N, dt, 1), matrices(1, T, K, dt, 2)[0]
    R = T * per
    rng = np.random.default_rng(E)
    index = rng.integers(0, E, R)
    index[rng.random(R) < 0.2] = -1            # rows without an expert
    index[0] = E - 1
    idx = torch.tensor(index, dtype=torch.int32, device="cuda")
    y = torch.full((R, N), 7.0, dtype=dt, device="cuda")
    with on_stream():
        Q, S = packed(w, group)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), buf(idx), buf(y), Q4Desc(group, 0)) == 0
    check_rows(x, quantised64(w, group), index.tolist(), y, group, torch.full_like(y, 7.0))


def test_gemv_all_rows_without_or_with_one_expert(lib):
    import torch
    w, x = matrices(3, 64, 32, torch.float16, 1), matrices(1, 20, 64, torch.float16, 2)[0]
    with on_stream():
        Q, S = packed(w, 64)
        for value in (-1, 2):
            idx = torch.full((20,), value, dtype=torch.int32, device="cuda")
            y = torch.full((20, 32), 7.0, dtype=torch.float32, device="cuda")
            assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), buf(idx), buf(y), Q4Desc(64, 0)) == 0
            check_rows(x, quantised64(w, 64), [value] * 20, y, 64, torch.full_like(y, 7.0))


def test_gemv_index_beyond_the_last_matrix(lib):
    import torch
    w, x = matrices(3, 64, 32, torch.bfloat16, 1), matrices(1, 4, 64, torch.bfloat16, 2)[0]
    index = [0, 3, 2 ** 31 - 1, 1]
    idx = torch.tensor(index, dtype=torch.int32, device="cuda")
    y = torch.full((4, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    with on_stream():
        Q, S = packed(w, 64)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), buf(idx), buf(y), Q4Desc(64, 0)) == -4
        check_rows(x, quantised64(w, 64), index, y, 64, torch.full_like(y, 7.0))
    with on_stream(asynchronous=True) as L:
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), buf(idx), buf(y), Q4Desc(64, 0)) == 0
        assert L.t2sp_b200_sync() == -4 and L.t2sp_b200_sync() == 0


@pytest.mark.parametrize("first,pad", [(0, 8), (1, 0), (1, 3), (8, 5)])
def test_gemv_strides(lib, first, pad):
    """Rows of x and y with a pitch, starting inside an allocation; what lies between the rows stays."""
    import torch
    R, K, N, group = 5, 200, 56, 64
    w = matrices(1, K, N, torch.bfloat16, 1)
    x0 = matrices(1, R, K, torch.bfloat16, 2)[0]
    bx = torch.full((R * (K + pad) + 64,), float("nan"), dtype=torch.bfloat16, device="cuda")
    by = torch.full((R * (N + pad) + 64,), 9.0, dtype=torch.bfloat16, device="cuda")
    x = bx[first:].as_strided((R, K), (K + pad, 1))
    y = by[first:].as_strided((R, N), (N + pad, 1))
    x.copy_(x0)
    y.zero_()
    with on_stream():
        Q, S = packed(w, group)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), None, buf(y), Q4Desc(group, 0)) == 0
    check_rows(x0, quantised64(w, group), None, y, group)
    y.fill_(9.0)
    assert (by == 9).all()


def test_pack_strides(lib):
    """Matrices that are parts of a larger tensor, both ways round."""
    import torch
    big = matrices(3, 90, 70, torch.float16, 4)
    part = big[1:3, 5:83, 3:60]
    for trans in (False, True):
        stored = part if not trans else big.transpose(1, 2).contiguous().transpose(1, 2)[1:3, 5:83, 3:60].transpose(1, 2)
        with on_stream():
            Q, S = packed(stored, 32, trans)
            out = torch.full((3, 80, 80), 5.0, dtype=torch.float16, device="cuda")
            view = out[:2, 1:1 + stored.shape[1], 2:2 + stored.shape[2]]
            assert t2sp_b200.q4_unpack(buf(Q), buf(S), buf(view), Q4Desc(32, int(trans))) == 0
        want = quantised64(part, 32).half()
        assert torch.equal(view.transpose(1, 2) if trans else view, want)
        view.fill_(5.0)
        assert (out == 5).all()


def test_gemv_empty_contraction(lib):
    import torch
    y = torch.full((2, 24), 7.0, dtype=torch.bfloat16, device="cuda")
    X = Buffer((0, 2), "bf16", host=y.data_ptr())
    Q = Buffer((512, 0, 2, 1), "u8", host=y.data_ptr())
    S = Buffer((16, 0, 2, 1), "bf16", host=y.data_ptr())
    with on_stream():
        assert t2sp_b200.q4_gemv(X, Q, S, None, buf(y), Q4Desc(64, 0)) == 0
    assert not y.any()


def test_host_buffers(lib):
    import torch
    w = matrices(2, 70, 20, torch.float16, 3)
    x = matrices(1, 3, 70, torch.float16, 4)[0]
    W, X = Buffer.from_numpy(w.cpu().numpy()), Buffer.from_numpy(x.cpu().numpy())
    q, s = Buffer.query(4, "u8"), Buffer.query(4, "f16")
    assert t2sp_b200.q4_pack(W, q, s, Q4Desc(32, 0)) == 0
    Q = Buffer.from_numpy(np.zeros([e for _, e, _ in reversed(q.shape())], np.uint8))
    S = Buffer.from_numpy(np.zeros([e for _, e, _ in reversed(s.shape())], np.float16))
    Y = Buffer.from_numpy(np.full((3, 20), 7.0, np.float32))
    assert t2sp_b200.q4_pack(W, Q, S, Q4Desc(32, 0)) == 0
    assert t2sp_b200.q4_gemv(X, Q, S, Buffer.from_numpy(np.array([1, -1, 0], np.int32)), Y, Q4Desc(32, 0)) == 0
    y = torch.from_numpy(Y.keepalive).cuda()
    check_rows(x, quantised64(w, 32), [1, -1, 0], y, 32, torch.full_like(y, 7.0))


def test_experts_of_a_layer_together(lib):
    """A layer's experts as a host program uses them: a training step with the grouped products, the weights quantised once, a prompt
    with the values read back, and single tokens from the packed form, captured into a graph and replayed; both give the prompt's rows."""
    import torch
    E, K, N, group, dt = 6, 192, 320, 64, torch.bfloat16
    w = matrices(E, K, N, dt, 1, K ** -0.5)
    counts = [9, 0, 30, 1, 64, 12]
    M = sum(counts)
    off = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    x = matrices(1, M, K, dt, 2)[0]
    d = matrices(1, M, N, dt, 3)[0]
    dx, dw = torch.empty_like(x), torch.empty(E, K, N, dtype=torch.float32, device="cuda")
    prompt = torch.empty(M, N, dtype=torch.float32, device="cuda")
    with on_stream(asynchronous=True) as L:
        assert t2sp_b200.grouped_gemm(buf(d), buf(w), buf(off), buf(dx), GroupedDesc(1)) == 0
        assert t2sp_b200.grouped_gemm_grad(buf(x), buf(d), buf(off), buf(dw)) == 0
        w -= (0.01 * dw).to(dt)                                        # on the same stream
        Q, S = packed(w, group)
        back = unpacked(Q, S, w, group)
        assert t2sp_b200.grouped_gemm(buf(x), buf(back), buf(off), buf(prompt)) == 0
        assert L.t2sp_b200_sync() == 0
    expert = torch.repeat_interleave(torch.arange(E), torch.tensor(counts)).to(torch.int32).cuda()
    pick = torch.tensor([M - 1, 0, 9, 39, 40, 38], device="cuda")
    token, index = x[pick].contiguous(), expert[pick].contiguous()
    y = torch.zeros(6, N, dtype=torch.float32, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    T, I, Y, QB, SB = (buf(t) for t in (token, index, y, Q, S))
    torch.cuda.synchronize()
    with on_stream(side, asynchronous=True):
        assert t2sp_b200.q4_gemv(T, QB, SB, I, Y, Q4Desc(group, 0)) == 0
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            rc = t2sp_b200.q4_gemv(T, QB, SB, I, Y, Q4Desc(group, 0))
    assert rc == 0
    for rows in (pick, torch.tensor([3, 50, 51, 100, 8, 7], device="cuda")):
        token.copy_(x[rows])
        index.copy_(expert[rows])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_rows(token, quantised64(w, group), index.tolist(), y, group)
        # the prompt used values rounded to bf16: half a step of 2^-8 of each product's magnitude
        mag = torch.stack([token[i].double().abs() @ back[index[i]].double().abs() for i in range(6)])
        assert ((y.double() - prompt[rows].double()).abs() <= mag * (eps_half(dt) + 64 * 2.0 ** -23)).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R", [1, 4, 8])
def test_gemv_ranges_of_x(lib, R, dtype):
    """Rows of x over the whole range of their type: outliers, numbers near the largest and the smallest, zeros, subnormal numbers.
    A value may be held to 2^-31 of the largest one in its row: that is added to the tolerance."""
    import torch
    dt = getattr(torch, dtype)
    fi = torch.finfo(dt)
    K, N, group = 448, 48, 64
    w = matrices(1, K, N, dt, 1, 1e-3)
    x = matrices(1, R, K, dt, 2)[0].float()
    x[:, 0:64] *= 2.0 ** -30 if dt == torch.bfloat16 else 2.0 ** -14
    x[:, 70] = 1000.0
    x[:, 128:192] = 0
    x[:, 192:256] = float(fi.max) * 2.0 ** -12 * torch.sign(x[:, 192:256])
    x[:, 256:320] = fi.smallest_normal * torch.sign(x[:, 256:320])
    x[:, 320:384] = fi.smallest_normal * fi.eps * torch.sign(x[:, 320:384])
    x = x.to(dt)
    y = torch.empty(R, N, dtype=torch.float32, device="cuda")
    for part in (slice(0, 192), slice(192, 256), slice(256, 448), slice(320, 384), slice(256, 320), slice(0, 448)):
        only = torch.zeros_like(x)
        only[:, part] = x[:, part]
        with on_stream():
            Q, S = packed(w, group)
            assert t2sp_b200.q4_gemv(buf(only), buf(Q), buf(S), None, buf(y), Q4Desc(group, 0)) == 0
        v, u = only.double(), quantised64(w, group)[0]
        top = v.abs().amax(1, keepdim=True)
        tol = ((group // 16 + 16) + (K // group + 16)) * 2.0 ** -23 * (v.abs() @ u.abs())
        tol = tol + 2.0 ** -31 * top * u.abs().sum(0) + 2.0 ** -140
        assert ((y.double() - v @ u).abs() <= tol).all(), part


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R", [1, 8])
def test_gemv_infinities_and_nan_of_x(lib, R, dtype):
    """A value of x that is not finite leaves nothing finite in its row; the other rows are as ever."""
    import torch
    dt = getattr(torch, dtype)
    w, x = matrices(1, 192, 40, dt, 1), matrices(1, R, 192, dt, 2)[0]
    bad = x.clone()
    bad[R - 1, 100] = float("inf")
    if R > 1:
        bad[2, 5] = float("nan")
    y = torch.empty(R, 40, dtype=torch.float32, device="cuda")
    with on_stream():
        Q, S = packed(w, 64)
        assert t2sp_b200.q4_gemv(buf(bad), buf(Q), buf(S), None, buf(y), Q4Desc(64, 0)) == 0
    hit = ~bad.isfinite().all(1)
    assert not y[hit].isfinite().any()
    if R > 1:
        rows = (~hit).nonzero().flatten()
        check_rows(x[rows], quantised64(w, 64), None, y[rows], 64)


@pytest.mark.parametrize("R,E,skip", [(1, 1, 1), (1, 1, 2), (4, 1, 1), (8, 1, 1), (16, 1, 2), (20, 7, 1)])
def test_gemv_bounded_waits_run_out(lib, R, E, skip):
    """Without one of the weights' copies (a test hook) the waits for it run out after the shortened limit, the kernel returns by itself, the
    call reports it, and the next call is right."""
    import torch
    from tests.util import library_env
    K, N, group = 4096, 4096, 64
    w, x = matrices(E, K, N, torch.bfloat16, 1), matrices(1, R, K, torch.bfloat16, 2)[0]
    index = [i % E for i in range(R)]
    idx = torch.tensor(index, dtype=torch.int32, device="cuda") if E > 1 else None
    y = torch.zeros(R, N, dtype=torch.float32, device="cuda")
    with on_stream():
        Q, S = packed(w, group)

        def call():
            return t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), buf(idx) if idx is not None else None, buf(y), Q4Desc(group, 0))
        with library_env(T2SP_B200_WAIT_CYCLES="20000000", T2SP_B200_TEST_SKIP_STAGE=str(skip)):
            assert call() == -23
        assert call() == 0
    check_rows(x, quantised64(w, group), index, y, group)


def spread_rows(R, K, dtype, seed=2):
    """Rows of x whose even ones hold a value so large, at k = 5, that 31 bits from it down do not reach the others."""
    import torch
    x = matrices(1, R, K, dtype, seed)[0]
    x[::2] *= 2.0 ** -30 if dtype == torch.bfloat16 else 2.0 ** -11
    x[::2, 5] = 1000.0 if dtype == torch.bfloat16 else 60000.0
    return x


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,K,N,group", [(1, 448, 48, 64), (2, 300, 33, 32), (2, 1000, 70, 128), (3, 192, 40, 64), (4, 448, 48, 32), (4, 700, 48, 128), (8, 448, 48, 64),
                                         (4, 7500, 24, 64), (4, 8192, 24, 64), (1, 30000, 20, 64), (1, 33000, 20, 64), (5, 65, 17, 128)])
def test_gemv_large_values_that_meet_zeros(lib, R, K, N, group, dtype):
    """Where the row's largest value meets a zero of W, the others are the whole result: it is as exact as any. Both sides of the lengths
    up to which a few rows are held as integers (4 rows: about 7900 values, 1 row: about 31000). Rows beside are the same to the bit."""
    import torch
    dt = getattr(torch, dtype)
    w = matrices(1, K, N, dt, 1)
    w[0, 5, ::2] = 0
    x = spread_rows(R, K, dt)
    plain = x.clone()
    plain[::2] = matrices(1, R, K, dt, 5)[0][::2]
    y, z = (torch.empty(R, N, dtype=torch.float32, device="cuda") for _ in range(2))
    with on_stream():
        Q, S = packed(w, group)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), None, buf(y), Q4Desc(group, 0)) == 0
        assert t2sp_b200.q4_gemv(buf(plain), buf(Q), buf(S), None, buf(z), Q4Desc(group, 0)) == 0
    check_rows(x, quantised64(w, group), None, y, group)
    check_rows(plain, quantised64(w, group), None, z, group)
    assert torch.equal(y[1::2], z[1::2])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_gemv_large_values_by_expert(lib, dtype):
    import torch
    dt = getattr(torch, dtype)
    E, T, per, K, N, group = 5, 7, 2, 320, 50, 64
    w, x = matrices(E, K, N, dt, 1), spread_rows(T, K, dt)
    w[:, 5, ::2] = 0
    index = [3, 1, 3, 3, -1, 0, 3, 4, 3, 3, 2, 1, 1, 0]
    idx = torch.tensor(index, dtype=torch.int32, device="cuda")
    y = torch.full((T * per, N), 7.0, dtype=torch.float32, device="cuda")   # the large products leave f16
    with on_stream():
        Q, S = packed(w, group)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), buf(idx), buf(y), Q4Desc(group, 0)) == 0
    check_rows(x, quantised64(w, group), index, y, group, torch.full_like(y, 7.0))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("R,K", [(1, 192), (2, 192), (4, 320), (8, 192), (4, 8192), (1, 33000)])
def test_gemv_infinities_of_x_follow_the_products(lib, R, K, dtype):
    """inf * q is an infinity of q's sign, and NaN where q is 0; infinities of both signs give NaN; the other rows are as ever."""
    import torch
    dt = getattr(torch, dtype)
    w, x = matrices(1, K, 40, dt, 1), matrices(1, R, K, dt, 2)[0]
    x[0, 100] = float("inf")
    if R > 1:
        x[1, 7], x[1, 90] = -float("inf"), float("inf")
    if R > 3:
        x[3, 3] = float("nan")
    y = torch.empty(R, 40, dtype=torch.float32, device="cuda")
    values = quantised64(w, 64)
    with on_stream():
        Q, S = packed(w, 64)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), None, buf(y), Q4Desc(64, 0)) == 0
    for r in range(R):
        want = (x[r].double()[:, None] * values[0]).sum(0)
        if x[r].isfinite().all():
            check_rows(x[r:r + 1], values, None, y[r:r + 1], 64)
        else:
            assert not want.isfinite().any() and torch.equal(y[r].double().nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("rows,K,N,pad", [(1, 256, 512, 0), (8, 256, 512, 3), (160, 515, 1031, 0)])
def test_results_of_one_call_are_the_next_ones_operand(lib, rows, K, N, pad):
    """Asynchronous calls on one stream, each reading at once what the one before writes: rows for q4_gemv, B with rows off 16 bytes
    for the grouped product. Two sets of inputs in turn, so that what an earlier round left would show; equal to synchronous calls."""
    import torch
    from tests.device_util import packed as pack
    dt = torch.bfloat16
    E, group = 8, 64
    sets = [matrices(1, rows, K, dt, s)[0] for s in (1, 2)]
    ds = [matrices(1, rows, N, dt, s)[0] for s in (3, 4)]
    w, b = matrices(1, N, 96, dt, 5), matrices(E, K, N, dt, 6, K ** -0.5)
    off = torch.tensor([i * rows // E for i in range(E + 1)], dtype=torch.int32, device="cuda")
    mid = torch.zeros(rows, N + pad, dtype=dt, device="cuda")[:, :N]
    g = torch.zeros(E, K, N, dtype=dt, device="cuda")
    out = torch.zeros(rows, N, dtype=dt, device="cuda")
    y = torch.zeros(rows, 96, dtype=torch.float32, device="cuda")

    def chain(i, L=None):
        assert t2sp_b200.grouped_gemm_grad(buf(sets[i]), buf(ds[i]), buf(off), buf(g)) == 0
        assert t2sp_b200.grouped_gemm(buf(sets[1 - i]), buf(g), buf(off), buf(out)) == 0
        assert t2sp_b200.grouped_gemm(buf(sets[i]), buf(b), buf(off), buf(mid)) == 0
        assert t2sp_b200.q4_gemv(buf(mid), buf(Q), buf(S), None, buf(y), Q4Desc(group, 0)) == 0
    with on_stream():
        Q, S = pack(w, group)
        want = []
        for i in (0, 1):
            chain(i)
            want.append([t.clone() for t in (g, out, mid, y)])
        check_rows(want[1][2], quantised64(w, group), None, want[1][3], group)
    keep = []
    with on_stream(asynchronous=True) as L:
        for n in range(40):
            chain(n % 2)
            if n >= 30:
                keep.append((n % 2, [t.clone() for t in (g, out, mid, y)]))
        assert L.t2sp_b200_sync() == 0
    for i, got in keep:
        assert all(torch.equal(a, b) for a, b in zip(got, want[i]))


@pytest.mark.parametrize("R,indexed", [(1, False), (2, True), (5, False), (17, True)])
def test_gemv_of_no_k(lib, R, indexed):
    """K = 0: the sums are empty, the results zeros, in every form of the product; a row without a matrix is left as it was."""
    import torch
    N, E = 24, 2 if indexed else 1
    y = torch.full((R, N), 7.0, dtype=torch.float32, device="cuda")
    index = torch.tensor([(i % 3) - 1 for i in range(R)], dtype=torch.int32, device="cuda")
    X = Buffer((0, R), "f16", host=y.data_ptr())       # nothing of an empty operand is read
    Q = Buffer((512, 0, 2, E), "u8", host=y.data_ptr())
    S = Buffer((16, 0, 2, E), "f16", host=y.data_ptr())
    with on_stream():
        assert t2sp_b200.q4_gemv(X, Q, S, buf(index) if indexed else None, buf(y), Q4Desc(32, 0)) == 0
    left = (index < 0) if indexed else torch.zeros(R, dtype=torch.bool, device="cuda")
    assert (y[left] == 7).all() and not y[~left].any()


@pytest.mark.parametrize("R", [1, 2, 4, 8])
@pytest.mark.parametrize("w_scale,x_scale", [(2.0 ** 122, 2.0 ** -40), (2.0 ** 122, 2.0 ** -120), (2.0 ** 60, 2.0 ** 50), (2.0 ** -110, 2.0 ** 90), (2.0 ** -60, 2.0 ** -60),
                                             (2.0 ** 100, 2.0 ** -75), (2.0 ** 10, 2.0 ** -126)])
def test_gemv_ranges_of_w_and_x(lib, R, w_scale, x_scale):
    """Large matrices times small rows and the other way round, over bf16's range: finite wherever the result is, and as exact as any (sums below
    fp32's smallest normal number 2^-126 have steps of 2^-149)."""
    import torch
    K, N, group = 448, 48, 64
    w = (matrices(1, K, N, torch.float32, 1).clamp(-8, 8) * w_scale).bfloat16()
    x = (matrices(1, R, K, torch.float32, 2)[0] * x_scale).bfloat16()
    assert w.isfinite().all()
    y = torch.empty(R, N, dtype=torch.float32, device="cuda")
    with on_stream():
        Q, S = packed(w, group)
        assert t2sp_b200.q4_gemv(buf(x), buf(Q), buf(S), None, buf(y), Q4Desc(group, 0)) == 0
    v, u = x.double(), quantised64(w, group)[0]
    tol = ((group // 16 + 16) + (K // group + 16)) * 2.0 ** -23 * (v.abs() @ u.abs()) + 2.0 ** -140
    assert ((y.double() - v @ u).abs() <= tol).all()
