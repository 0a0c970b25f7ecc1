"""Device-resident calls for the tests: torch tensors as buffers of the library, on torch's current stream."""
import contextlib
import ctypes

import t2sp_b200
from t2sp_b200 import Buffer


def names():
    import torch
    return {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32", torch.int32: "i32", torch.uint8: "u8"}


def buf(t):
    """The tensor's memory as a buffer (torch's last dimension is dimension 0)."""
    b = Buffer(tuple(reversed(t.shape)), names()[t.dtype], strides=tuple(reversed(t.stride())), keepalive=t)
    assert t2sp_b200.wrap_device(b, t.data_ptr()) == 0
    return b


@contextlib.contextmanager
def on_stream(stream=None, asynchronous=False):
    """Calls of this thread go to `stream` (torch's current one by default)."""
    import torch
    L = t2sp_b200.lib()
    handle = (stream if stream is not None else torch.cuda.current_stream()).cuda_stream or 1   # 1: the legacy default stream
    L.t2sp_b200_set_stream(ctypes.c_void_p(handle))
    L.t2sp_b200_set_async(1 if asynchronous else 0)
    try:
        yield L
    finally:
        L.t2sp_b200_set_async(0)
        L.t2sp_b200_set_stream(None)


def eps_half(dtype):
    """A rounding to `dtype` is off by at most this, relative to the value."""
    import torch
    return torch.finfo(dtype).eps / 2


def packed(w, group=64, trans=False):
    """(Q, S) tensors of the quantised w: (E, K, N), or (E, N, K) with trans."""
    import torch
    desc = t2sp_b200.Q4Desc(group, 1 if trans else 0)
    q, s = Buffer.query(4, "u8"), Buffer.query(4, names()[w.dtype])
    assert t2sp_b200.q4_pack(buf(w), q, s, desc) == 0
    Q = torch.zeros([e for _, e, _ in reversed(q.shape())], dtype=torch.uint8, device=w.device)
    S = torch.zeros([e for _, e, _ in reversed(s.shape())], dtype=w.dtype, device=w.device)
    assert t2sp_b200.q4_pack(buf(w), buf(Q), buf(S), desc) == 0
    return Q, S


def quantised64(w, group):
    """The values that the 4-bit form of w (E, K, N) stands for, and the scales, in 64 bits."""
    import torch
    E, K, N = w.shape
    out = torch.zeros(E, K, N, dtype=torch.float64, device=w.device)
    for k in range(0, K, group):
        part = w[:, k:k + group].double()
        s = (part.abs().amax(1, keepdim=True) / 7).to(w.dtype).double()
        q = torch.where(s > 0, torch.round(part / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(part))
        out[:, k:k + group] = q.clamp(-7, 7) * s
    return out
