"""Refusals and bounds queries of the grouped and the 4-bit products: nothing here needs a GPU (a valid call ends with
-36, no device, where there is none)."""
import numpy as np
import pytest

import t2sp_b200
from t2sp_b200 import Buffer, GroupedDesc, Q4Desc


def no_device():
    import torch
    return not torch.cuda.is_available()


def h16(*shape, dtype="bf16"):
    return Buffer.from_numpy(np.zeros(shape, np.uint16), dtype=dtype)


def i32(*shape):
    return Buffer.from_numpy(np.zeros(shape, np.int32))


def f32(*shape):
    return Buffer.from_numpy(np.zeros(shape, np.float32))


def grouped(M=8, K=16, N=24, E=3, **kw):
    a = dict(A=h16(M, K), B=h16(E, K, N), offsets=i32(E + 1), C=h16(M, N))
    a.update(kw)
    return t2sp_b200.grouped_gemm(a["A"], a["B"], a["offsets"], a["C"], a.get("desc"))


def grad(M=8, K=16, N=24, E=3, **kw):
    a = dict(A=h16(M, K), D=h16(M, N), offsets=i32(E + 1), G=h16(E, K, N))
    a.update(kw)
    return t2sp_b200.grouped_gemm_grad(a["A"], a["D"], a["offsets"], a["G"])


def strided(extents, strides, dtype="bf16"):
    return Buffer(extents, dtype, host=np.zeros(1 << 16, np.uint16).ctypes.data, strides=strides)


def test_grouped_null_and_types(lib):
    assert lib.t2sp_b200_grouped_gemm(None, None, None, None, None) == -12
    assert lib.t2sp_b200_grouped_gemm_grad(h16(1, 1).ptr, None, i32(2).ptr, h16(1, 1, 1).ptr) == -12
    assert grouped(A=f32(8, 16)) == -3                 # 16-bit operands only
    assert grouped(B=h16(3, 16, 24, dtype="f16")) == -3   # one type for A and B
    assert grouped(C=h16(8, 24, dtype="f16")) == -3
    assert grouped(offsets=f32(4)) == -3
    assert grouped(B=h16(16, 24)) == -43
    assert grad(G=h16(16, 24)) == -43
    assert grad(D=h16(8, 24, dtype="f16")) == -3


def test_grouped_shapes(lib):
    assert grouped(B=h16(3, 17, 24)) == -8             # K differs
    assert grouped(B=h16(3, 24, 16)) == -8
    if no_device():
        assert grouped(B=h16(3, 24, 16), desc=GroupedDesc(1)) == -36
        assert grouped(C=f32(8, 24)) == -36            # fp32 results too
        assert grad() == -36 and grad(G=Buffer.from_numpy(np.zeros((3, 16, 24), np.float32))) == -36
    assert grouped(offsets=i32(3)) == -8               # E + 1 offsets
    assert grouped(C=h16(7, 24)) == -4 and grouped(C=h16(8, 23)) == -4
    assert grad(D=h16(7, 24)) == -8
    assert grad(G=h16(2, 16, 24)) == -4 and grad(G=h16(3, 15, 24)) == -4
    assert grouped(E=1025) == -8                       # at most 1024 groups
    assert grad(offsets=i32(0)) == -8
    A = h16(8, 16)
    A.dims[1].extent = -1
    assert grouped(A=A) == -28
    A = h16(8, 16)
    A.dims[1].min = 2                                  # inputs start at 0
    assert grouped(A=A) == -4


def test_grouped_strides(lib):
    assert grouped(A=strided((16, 8), (2, 32))) == -8              # the innermost stride is 1
    assert grouped(A=strided((16, 8), (1, 0))) == -8               # rows at one address
    assert grouped(C=strided((24, 8), (1, 23))) == -8              # rows of the output overlap
    assert grad(G=strided((24, 16, 3), (1, 24, 24))) == -8
    if no_device():
        assert grouped(A=strided((16, 8), (1, 19))) == -36
        assert grad(G=strided((24, 16, 3), (1, 72, 24))) == -36     # matrices interleaved row by row


def test_grouped_empty_calls(lib):
    assert grouped(M=0) == 0 and grouped(N=0) == 0 and grouped(E=0, B=h16(0, 16, 24)) == 0
    assert grad(K=0, A=h16(8, 0), G=h16(3, 0, 24)) == 0
    assert grad(E=0, G=h16(0, 16, 24)) == 0


def test_grouped_bounds_queries(lib):
    q = Buffer.query(2)
    assert grouped(C=q) == 0 and [e for _, e, _ in q.shape()] == [24, 8] and q.raw.type.bits == 16
    q = Buffer.query(3)
    assert grad(G=q) == 0 and [e for _, e, _ in q.shape()] == [24, 16, 3]
    q, o = Buffer.query(3), Buffer.query(1)
    assert grouped(B=q, C=h16(8, 24), desc=GroupedDesc(1)) == 0 and [e for _, e, _ in q.shape()] == [16, 24, 3]
    assert grouped(offsets=o) == 0 and [e for _, e, _ in o.shape()] == [4]


def q4_args(N=40, K=100, E=2, R=6, T=3, group=32, dtype="bf16"):
    kb, nb = -(-K // 64), -(-N // 16)
    return dict(X=h16(T, K, dtype=dtype), Q=Buffer.from_numpy(np.zeros((E, nb, kb, 512), np.uint8)),
                S=h16(E, nb, -(-kb * 64 // group), 16, dtype=dtype), index=i32(R), Y=h16(R, N, dtype=dtype), desc=Q4Desc(group, 0))


def gemv(**kw):
    sizes = {k: kw.pop(k) for k in ("N", "K", "E", "R", "T", "group", "dtype") if k in kw}
    a = q4_args(**sizes)
    a.update(kw)
    return t2sp_b200.q4_gemv(a["X"], a["Q"], a["S"], a["index"], a["Y"], a["desc"])


def test_q4_queries(lib):
    for group, groups in ((32, 4), (64, 2), (128, 1)):
        q, s = Buffer.query(4), Buffer.query(4)
        assert t2sp_b200.q4_pack(h16(2, 100, 40), q, s, Q4Desc(group, 0)) == 0
        assert [e for _, e, _ in q.shape()] == [512, 2, 3, 2] and q.raw.type.bits == 8
        assert [e for _, e, _ in s.shape()] == [16, groups, 3, 2] and s.raw.type.bits == 16
    q, s = Buffer.query(4), Buffer.query(4)
    assert t2sp_b200.q4_pack(h16(2, 40, 100), q, s, Q4Desc(0, 1)) == 0     # k innermost, the default group of 64
    assert [e for _, e, _ in q.shape()] == [512, 2, 3, 2] and [e for _, e, _ in s.shape()] == [16, 2, 3, 2]


def test_q4_refusals(lib):
    a = q4_args()
    assert lib.t2sp_b200_q4_gemv(None, a["Q"].ptr, a["S"].ptr, None, a["Y"].ptr, None) == -12
    assert lib.t2sp_b200_q4_pack(None, a["Q"].ptr, a["S"].ptr, None) == -12
    assert lib.t2sp_b200_q4_unpack(a["Q"].ptr, a["S"].ptr, None, None) == -12
    assert gemv(desc=Q4Desc(48, 0)) == -8
    assert gemv(desc=Q4Desc(64, 0)) == -8              # the scales are those of groups of 32
    assert gemv(X=f32(3, 100)) == -3
    assert gemv(X=h16(3, 100, dtype="f16")) == -3      # X and S have one type
    assert gemv(Y=h16(6, 40, dtype="f16")) == -3
    assert gemv(index=None) == -8                      # several matrices and no index
    assert gemv(index=i32(5)) == -8
    assert gemv(T=4) == -8                             # 6 rows are no multiple of 4
    assert gemv(T=0) == -8
    assert gemv(Y=h16(6, 60)) == -8                    # the packed matrices have 48 columns at most
    assert gemv(X=h16(3, 130)) == -8
    assert gemv(Y=strided((40, 6), (1, 39))) == -8
    b = Buffer.from_numpy(np.zeros((2, 3, 2, 512), np.uint8))
    b.dims[1].stride = 513
    assert gemv(Q=b) == -8
    b = Buffer.from_numpy(np.zeros((2, 3, 2, 512), np.uint8))
    assert t2sp_b200.wrap_device(b, 4096 + 8) == 0     # the packed matrices start on 16 bytes
    assert gemv(Q=b) == -8
    assert gemv(R=0, T=1) == 0
    assert gemv(K=100000, N=16, E=1, R=1, T=1) == -8   # a row of x has to fit in shared memory
    assert gemv(R=1025, T=1025) == -8                  # rows that name their matrix: at most 1024
    if no_device():
        assert gemv() == -36 and gemv(E=1, index=None) == -36 and gemv(Y=f32(6, 40)) == -36
    W = h16(2, 100, 40)
    assert t2sp_b200.q4_pack(W, a["Q"], a["S"], Q4Desc(64, 0)) == -8
    assert t2sp_b200.q4_pack(Buffer.from_numpy(np.zeros((2, 100, 40), np.float32)), a["Q"], a["S"], Q4Desc(32, 0)) == -3
    assert t2sp_b200.q4_unpack(a["Q"], a["S"], h16(2, 40, 100), Q4Desc(32, 0)) == -8    # would need trans_b
    if no_device():
        assert t2sp_b200.q4_unpack(a["Q"], a["S"], h16(2, 40, 100), Q4Desc(32, 1)) == -36
        assert t2sp_b200.q4_pack(W, a["Q"], a["S"], Q4Desc(32, 0)) == -36


@pytest.mark.parametrize("name", ["grouped_gemm", "grouped_gemm_grad", "q4_pack", "q4_unpack", "q4_gemv"])
def test_no_device_launches_nothing(lib, name):
    if not no_device():
        pytest.skip("a GPU is present")
    before = lib.t2sp_b200_kernel_launches()
    a = q4_args()
    assert {"grouped_gemm": grouped, "grouped_gemm_grad": grad, "q4_gemv": gemv,
            "q4_pack": lambda: t2sp_b200.q4_pack(h16(2, 100, 40), a["Q"], a["S"], a["desc"]),
            "q4_unpack": lambda: t2sp_b200.q4_unpack(a["Q"], a["S"], h16(2, 100, 40), a["desc"])}[name]() == -36
    assert lib.t2sp_b200_kernel_launches() == before


def test_extent_limits(lib):
    # 32-bit counts: extents end at 2^30 (the packed shapes of such a matrix would not fit 32 bits either)
    big, top = (1 << 30) + 1, (1 << 31) - 1
    for n in (big, top):
        assert grouped(A=strided((16, n), (1, 16)), C=strided((24, n), (1, 24))) == -6
        assert grad(A=strided((n, 8), (1, n)), G=strided((24, n, 3), (1, 24, 24))) == -6
        assert gemv(X=strided((n, 3), (1, n))) == -6
        a = q4_args()
        assert t2sp_b200.q4_pack(strided((40, n, 2), (1, 40, 40)), a["Q"], a["S"], a["desc"]) == -6


def test_device_addresses(lib):
    def at(extents, dtype, address):
        b = Buffer(extents, dtype)
        assert t2sp_b200.wrap_device(b, address) == 0
        return b
    assert grouped(A=at((16, 8), "bf16", 4097)) == -8
    assert grouped(C=at((24, 8), "f32", 4098)) == -8
    assert grouped(offsets=at((4,), "i32", 4098)) == -8
    assert grad(G=at((24, 16, 3), "f32", 4098)) == -8
    assert gemv(X=at((100, 3), "bf16", 4097)) == -8
    assert gemv(Y=at((40, 6), "f32", 4098)) == -8
    assert gemv(index=at((6,), "i32", 4097)) == -8
    a = q4_args()
    assert t2sp_b200.q4_pack(at((40, 100, 2), "bf16", 4097), a["Q"], a["S"], a["desc"]) == -8
    assert t2sp_b200.q4_unpack(a["Q"], a["S"], at((40, 100, 2), "bf16", 4097), a["desc"]) == -8


def test_q4_bounds_queries_of_products_and_reading(lib):
    a = q4_args()
    q = Buffer.query(2)
    assert gemv(Y=Buffer.query(2)) == 0 and gemv(Y=q) == 0 and [e for _, e, _ in q.shape()] == [48, 6]
    q = Buffer.query(2)
    assert gemv(X=q) == 0 and [e for _, e, _ in q.shape()] == [128, 6] and q.raw.type.bits == 16
    q, s, i = Buffer.query(4), Buffer.query(4), Buffer.query(1)
    assert gemv(Q=q) == 0 and [e for _, e, _ in q.shape()] == [512, 2, 3, 1]
    assert gemv(S=s) == 0 and [e for _, e, _ in s.shape()] == [16, 4, 3, 2]
    assert gemv(index=i) == 0 and [e for _, e, _ in i.shape()] == [6]
    for trans in (0, 1):
        w = Buffer.query(3)
        assert t2sp_b200.q4_unpack(a["Q"], a["S"], w, Q4Desc(32, trans)) == 0
        assert [e for _, e, _ in w.shape()] == ([128, 48, 2] if trans else [48, 128, 2]) and w.raw.type.bits == 16
    assert t2sp_b200.q4_pack(Buffer.query(3), Buffer.query(4), Buffer.query(4)) == -34


def test_output_strides_of_matrices_that_interlock(lib):
    """An output's matrices may begin where the last row of the one before ends, not only a whole pitch later."""
    near, over = strided((24, 16, 3), (1, 32, 15 * 32 + 24), "f32"), strided((24, 16, 3), (1, 32, 15 * 32 + 23), "f32")
    assert grad(G=over) == -8
    if no_device():
        assert grad(G=near) == -36
        assert t2sp_b200.q4_unpack(q4_args()["Q"], q4_args()["S"], strided((40, 100, 2), (1, 48, 99 * 48 + 40)), Q4Desc(32, 0)) == -36


def test_bounds_queries_refuse_shapes_that_no_call_takes(lib):
    """Negative extents, extents beyond 2^30 and packed shapes whose matrix would have them give an error, not a shape."""
    a = q4_args()
    for extent, code in ((-1, -28), ((1 << 30) + 1, -6)):
        A = h16(8, 16)
        A.dims[1].extent = extent
        assert grouped(A=A, C=Buffer.query(2)) == code and grad(A=A, G=Buffer.query(3)) == code
        X = h16(3, 100)
        X.dims[1].extent = extent
        assert gemv(X=X, Y=Buffer.query(2)) == code
        W = h16(2, 100, 40)
        W.dims[0].extent = extent
        assert t2sp_b200.q4_pack(W, Buffer.query(4), Buffer.query(4), a["desc"]) == code
        Q = q4_args()["Q"]
        Q.dims[2].extent = extent
        assert t2sp_b200.q4_unpack(Q, a["S"], Buffer.query(3), a["desc"]) == code
        assert gemv(Q=Q, X=Buffer.query(2)) == code
    for d, n in ((1, 1 << 25), (2, 1 << 28)):   # K or N of 2^31 and 2^32
        Q = q4_args()["Q"]
        Q.dims[d].extent = n
        assert t2sp_b200.q4_unpack(Q, a["S"], Buffer.query(3), a["desc"]) == -6
        assert gemv(Q=Q, X=Buffer.query(2), Y=Buffer.query(2)) == -6
    assert grouped(offsets=i32(0), B=Buffer.query(3)) == -8 and grad(offsets=i32(0), G=Buffer.query(3)) == -8
