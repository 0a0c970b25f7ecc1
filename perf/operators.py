"""Cases that measure the products grouped by expert and the 4-bit products of t2sp_b200.

Four operators, one pass of each as a host program makes it:

  forward    C[t] = A[t] x B[e(t)] for rows sorted by expert               (grouped_gemm)
  backward   the gradients of both operands of that product                (grouped_gemm with trans_b, grouped_gemm_grad)
  quantise   16-bit matrices to 4 bits with group scales, and read back    (q4_pack, q4_unpack)
  single     a few rows times 4-bit matrices, each row its own expert's    (q4_gemv)

With `own` false the same results come from elementary torch operations in 32 bits."""
import ctypes
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a handful of rows in decoding: the call's latency counts
        {"name": "forward few rows", "op": "forward", "E": 8, "T": 16, "K": 1024, "N": 1024, "dtype": "bf16", "trans": False, "skew": 0.0, "behind": 0},
        # decoding a batch: a few rows for each expert, every matrix is read once
        {"name": "forward decode", "op": "forward", "E": 64, "T": 256, "K": 2048, "N": 4096, "dtype": "bf16", "trans": False, "skew": 0.0, "behind": 0},
        # a long prompt or a training batch: bound by the matrix units
        {"name": "forward large", "op": "forward", "E": 8, "T": 16384, "K": 4096, "N": 8192, "dtype": "bf16", "trans": False, "skew": 0.3, "behind": 0},
        # a padded batch with uneven and empty groups, matrices stored transposed
        {"name": "forward ragged", "op": "forward", "E": 40, "T": 5003, "K": 1000, "N": 2040, "dtype": "f16", "trans": True, "skew": 1.5, "behind": 61},
        # the backward pass of a training step, both gradients
        {"name": "backward large", "op": "backward", "E": 8, "T": 16384, "K": 4096, "N": 4096, "dtype": "bf16", "skew": 0.3, "behind": 0},
        # a small step with uneven and empty groups
        {"name": "backward ragged", "op": "backward", "E": 24, "T": 1777, "K": 776, "N": 1416, "dtype": "f16", "skew": 1.5, "behind": 23},
        # one token, one matrix: latency counts
        {"name": "single one row", "op": "single", "E": 1, "T": 1, "R": 1, "K": 4096, "N": 4096, "G": 64, "dtype": "bf16"},
        # one token, a wide output: bound by memory
        {"name": "single wide", "op": "single", "E": 1, "T": 1, "R": 1, "K": 8192, "N": 32768, "G": 128, "dtype": "f16"},
        # eight tokens, two experts each
        {"name": "single experts", "op": "single", "E": 64, "T": 8, "R": 16, "K": 2048, "N": 4096, "G": 32, "dtype": "bf16"},
        # a small batch and odd sizes
        {"name": "single odd", "op": "single", "E": 1, "T": 13, "R": 13, "K": 1001, "N": 777, "G": 32, "dtype": "f16"},
        # a checkpoint's matrices, quantised and read back
        {"name": "quantise large", "op": "quantise", "E": 8, "K": 4096, "N": 4096, "G": 64, "dtype": "bf16", "trans": False},
        {"name": "quantise odd", "op": "quantise", "E": 3, "K": 1001, "N": 777, "G": 128, "dtype": "f16", "trans": True},
    ]


def _size(rng, lo, hi):
    n = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    step = rng.choice((64, 64, 8, 1))
    return max(lo, min(hi, int(round(n / step)) * step or step))


def draw(rng):
    op = rng.choice(("forward", "backward", "quantise", "single"))
    case = {"op": op, "dtype": rng.choice(("bf16", "f16"))}
    K, N = _size(rng, 128, 8192), _size(rng, 128, 8192)
    E = int(round(math.exp(rng.uniform(0.0, math.log(64)))))
    while E * K * N > 1 << 29:
        E = max(1, E // 2) if E > 1 else 1
        if E == 1:
            break
    if op in ("forward", "backward"):
        T = _size(rng, 1, 16384)
        top = (1 << 38) if op == "forward" else (1 << 37)
        T = min(T, max(1, top // (K * N)))
        case.update(E=E, T=T, K=K, N=N, skew=rng.choice((0.0, 0.5, 1.5)), behind=rng.choice((0, 0, 37)))
        if op == "forward":
            case["trans"] = rng.random() < 0.5
    elif op == "single":
        E = rng.choice((1, E))
        per = rng.choice((1, 2, 4))
        T = _size(rng, 1, 16)
        while E > 1 and T * per * K * N > 1 << 28 and T > 1:
            T = T // 2
        per = per if E > 1 and T * per * K * N <= 1 << 28 else 1
        case.update(E=E, T=T, R=T * per, K=K, N=N, G=rng.choice((32, 64, 128)))
    else:
        while E * K * N > 1 << 27 and E > 1:
            E = E // 2
        case.update(E=E, K=K, N=N, G=rng.choice((32, 64, 128)), trans=rng.random() < 0.5)
    return case


def _groups(case, gen):
    """Offsets of the experts' rows, as a router's choices give them, and the largest group."""
    E, T = case["E"], case["T"]
    logits = torch.randn(E, generator=gen, device="cuda") * case["skew"]
    expert = torch.multinomial(torch.softmax(logits, 0), T, replacement=True, generator=gen)
    counts = torch.bincount(expert, minlength=E)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = torch.cumsum(counts, 0)
    return offsets, int(counts.max())


def _buffer(t, dtype):
    """The host program's buffer of a tensor in device memory; dimension 0 is the innermost."""
    import t2sp_b200
    b = t2sp_b200.Buffer(tuple(reversed(t.shape)), dtype, strides=tuple(reversed(t.stride())), keepalive=t)
    t2sp_b200.wrap_device(b, t.data_ptr())
    return b


def _query(dims, dtype):
    import t2sp_b200
    return t2sp_b200.Buffer.query(dims, dtype)


def _alloc(q, dtype):
    """Device memory of the shape that a bounds query gave."""
    t = torch.empty([e for _, e, _ in reversed(q.shape())], dtype=dtype, device="cuda")
    return t


def _done(rc):
    if rc:
        raise RuntimeError("t2sp_b200 returned %d" % rc)


def _quantised(w, G):
    """(q, s): q in -7..7, one scale for G values along K; w is (E, K, N)."""
    E, K, N = w.shape
    groups = -(-K // G)
    padded = torch.nn.functional.pad(w.float(), (0, 0, 0, groups * G - K)).view(E, groups, G, N)
    s = (padded.abs().amax(2) / 7).to(w.dtype)
    wide = s.float().unsqueeze(2)
    q = torch.where(wide > 0, torch.round(padded / torch.where(wide > 0, wide, torch.ones_like(wide))), torch.zeros_like(padded))
    return q.clamp(-7, 7).view(E, groups * G, N)[:, :K], s


def _packed(w, G, trans):
    """The packed form of w and its scales as a host program keeps them: (tensors, buffers)."""
    import t2sp_b200
    desc = t2sp_b200.Q4Desc(G, 1 if trans else 0)
    name = "bf16" if w.dtype == torch.bfloat16 else "f16"
    wb, qb, sb = _buffer(w, name), _query(4, "u8"), _query(4, name)
    _done(t2sp_b200.q4_pack(wb, qb, sb, desc))
    q, s = _alloc(qb, torch.uint8), _alloc(sb, w.dtype)
    return (q, s), (_buffer(q, "u8"), _buffer(s, name)), desc


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    op, E, K, N = case["op"], case["E"], case["K"], case["N"]
    state = {"op": op}
    if own:
        # the calls go to torch's stream and return once they are enqueued
        import t2sp_b200
        lib = t2sp_b200.lib()
        lib.t2sp_b200_set_stream(ctypes.c_void_p(torch.cuda.current_stream().cuda_stream or 1))
        lib.t2sp_b200_set_async(1)
    name = case["dtype"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dt)

    if op in ("forward", "backward"):
        rows = case["T"] + case["behind"]
        offsets, capacity = _groups(case, gen)
        a = normal(rows, K)
        trans = bool(case.get("trans"))
        b = normal(E, N, K, scale=K ** -0.5) if trans else normal(E, K, N, scale=K ** -0.5)
        state.update(a=a, b=b, offsets=offsets, capacity=capacity, total=case["T"], trans=trans)
        if op == "forward":
            state["c"] = torch.zeros(rows, N, dtype=dt, device="cuda")
        else:
            state["dc"] = normal(rows, N)
            state["da"] = torch.zeros(rows, K, dtype=dt, device="cuda")
            state["db"] = torch.zeros(E, K, N, dtype=dt, device="cuda")
        if own:
            state["buffers"] = {k: _buffer(state[k], name) for k in ("a", "b", "c", "dc", "da", "db") if k in state}
            state["buffers"]["offsets"] = _buffer(offsets, "i32")
            state["desc"] = t2sp_b200.GroupedDesc(1 if trans or op == "backward" else 0)
    elif op == "single":
        w = normal(E, K, N, scale=K ** -0.5)
        x = normal(case["T"], K)
        index = torch.randint(0, E, (case["R"],), generator=gen, device="cuda", dtype=torch.int32) if E > 1 else None
        state.update(x=x, index=index, G=case["G"], y=torch.zeros(case["R"], N, dtype=dt, device="cuda"))
        if own:
            state["packed"], (qb, sb), state["desc"] = _packed(w, case["G"], False)
            _done(t2sp_b200.q4_pack(_buffer(w, name), qb, sb, state["desc"]))
            state["buffers"] = {"x": _buffer(x, name), "q": qb, "s": sb, "y": _buffer(state["y"], name),
                                "index": _buffer(index, "i32") if index is not None else None}
        else:
            q, s = _quantised(w, case["G"])
            state.update(q=q.to(torch.int8), s=s)
    else:
        trans = case["trans"]
        w = normal(E, N, K, scale=K ** -0.5) if trans else normal(E, K, N, scale=K ** -0.5)
        state.update(w=w, G=case["G"], trans=trans, back=torch.zeros_like(w))
        if own:
            state["packed"], (qb, sb), state["desc"] = _packed(w, case["G"], trans)
            state["buffers"] = {"w": _buffer(w, name), "q": qb, "s": sb, "back": _buffer(state["back"], name)}
    return state


def _places(state):
    """For each row that a group holds, its expert and its place in the group."""
    t = torch.arange(state["total"], device="cuda")
    offsets = state["offsets"].long()
    expert = torch.searchsorted(offsets[1:].contiguous(), t, right=True)
    return expert, t - offsets[expert]


def _padded(rows, expert, place, state):
    p = torch.zeros(state["offsets"].numel() - 1, state["capacity"], rows.shape[1], device="cuda")
    p[expert, place] = rows[: state["total"]].float()
    return p


def _scaled(q, s, G):
    """Values of 4-bit integers (.., K, N) with scales (.., groups, N)."""
    return q.float() * s.float().repeat_interleave(G, dim=-2)[..., : q.shape[-2], :]


def run(state):
    op = state["op"]
    if own:
        import t2sp_b200
        b = state["buffers"]
        if op == "forward":
            _done(t2sp_b200.grouped_gemm(b["a"], b["b"], b["offsets"], b["c"], state["desc"]))
            return state["c"]
        if op == "backward":
            _done(t2sp_b200.grouped_gemm(b["dc"], b["b"], b["offsets"], b["da"], state["desc"]))
            _done(t2sp_b200.grouped_gemm_grad(b["a"], b["dc"], b["offsets"], b["db"]))
            return state["da"], state["db"]
        if op == "single":
            _done(t2sp_b200.q4_gemv(b["x"], b["q"], b["s"], b["index"], b["y"], state["desc"]))
            return state["y"]
        _done(t2sp_b200.q4_pack(b["w"], b["q"], b["s"], state["desc"]))
        _done(t2sp_b200.q4_unpack(b["q"], b["s"], b["back"], state["desc"]))
        return state["back"]
    if op == "forward":
        expert, place = _places(state)
        b = state["b"].float()
        c = torch.bmm(_padded(state["a"], expert, place, state), b.transpose(1, 2) if state["trans"] else b)
        state["c"][: state["total"]] = c[expert, place].to(state["c"].dtype)
        return state["c"]
    if op == "backward":
        expert, place = _places(state)
        a, dc = (_padded(state[k], expert, place, state) for k in ("a", "dc"))
        da = torch.bmm(dc, state["b"].float().transpose(1, 2))
        state["da"][: state["total"]] = da[expert, place].to(state["da"].dtype)
        state["db"].copy_(torch.bmm(a.transpose(1, 2), dc))
        return state["da"], state["db"]
    if op == "single":
        x, q, s = state["x"].float(), state["q"], state["s"]
        if state["index"] is None:
            y = x @ _scaled(q[0], s[0], state["G"])
        else:
            e = state["index"].long()
            x = x.repeat_interleave(e.numel() // x.shape[0], dim=0)
            y = torch.bmm(x.unsqueeze(1), _scaled(q[e], s[e], state["G"])).squeeze(1)
        state["y"].copy_(y)
        return state["y"]
    w = state["w"].transpose(1, 2) if state["trans"] else state["w"]
    q, s = _quantised(w, state["G"])
    back = _scaled(q, s, state["G"])
    state["back"].copy_(back.transpose(1, 2) if state["trans"] else back)
    return state["back"]


def work(case):
    E, K, N = case["E"], case["K"], case["N"]
    if case["op"] == "quantise":
        packed = K * N / 2 + -(-K // case["G"]) * N * 2
        return {"bytes": E * (4 * K * N + 2 * packed), "flops": E * K * N}
    if case["op"] == "single":
        read = E * (1 - (1 - 1 / E) ** case["R"])  # matrices that the rows are expected to name
        packed = K * N / 2 + -(-K // case["G"]) * N * 2
        return {"bytes": read * packed + 2 * case["T"] * K + 2 * case["R"] * N, "flops": 2 * case["R"] * K * N}
    T = case["T"]
    read = E * (1 - (1 - 1 / E) ** T) if case["skew"] < 1 else min(E, T)
    if case["op"] == "forward":
        return {"bytes": 2 * (T * K + T * N + read * K * N), "flops": 2 * T * K * N}
    return {"bytes": 2 * (2 * T * K + T * N + read * K * N + E * K * N), "flops": 4 * T * K * N}


def exact(case, seed):
    """The same results in 64 bits, expert by expert."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    op, E, K, N = case["op"], case["E"], case["K"], case["N"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dt)

    if op in ("forward", "backward"):
        rows = case["T"] + case["behind"]
        offsets = _groups(case, gen)[0].tolist()
        a = normal(rows, K)
        trans = bool(case.get("trans"))
        b = normal(E, N, K, scale=K ** -0.5) if trans else normal(E, K, N, scale=K ** -0.5)
        if op == "forward":
            c = torch.zeros(rows, N, dtype=torch.float64, device="cuda")
            for e in range(E):
                lo, hi = offsets[e], offsets[e + 1]
                c[lo:hi] = a[lo:hi].double() @ (b[e].double().T if trans else b[e].double())
            return c
        dc = normal(rows, N)
        da = torch.zeros(rows, K, dtype=torch.float64, device="cuda")
        db = torch.zeros(E, K, N, dtype=torch.float64, device="cuda")
        for e in range(E):
            lo, hi = offsets[e], offsets[e + 1]
            da[lo:hi] = dc[lo:hi].double() @ b[e].double().T
            db[e] = a[lo:hi].double().T @ dc[lo:hi].double()
        return da, db

    def values(w):  # one (K, N) matrix as its 4-bit form stands for it
        out = torch.empty(w.shape, dtype=torch.float64, device="cuda")
        for k in range(0, K, case["G"]):
            part = w[k : k + case["G"]].double()
            s = (part.abs().amax(0) / 7).to(dt).double()
            q = torch.where(s > 0, torch.round(part / s), torch.zeros_like(part)).clamp(-7, 7)
            out[k : k + case["G"]] = q * s
        return out

    if op == "single":
        w = normal(E, K, N, scale=K ** -0.5)
        x = normal(case["T"], K)
        index = torch.randint(0, E, (case["R"],), generator=gen, device="cuda", dtype=torch.int32).tolist() if E > 1 else [0] * case["R"]
        y = torch.zeros(case["R"], N, dtype=torch.float64, device="cuda")
        per = case["R"] // case["T"]
        for e in sorted(set(index)):
            at = [r for r in range(case["R"]) if index[r] == e]
            y[at] = x[[r // per for r in at]].double() @ values(w[e])
        return y
    trans = case["trans"]
    w = normal(E, N, K, scale=K ** -0.5) if trans else normal(E, K, N, scale=K ** -0.5)
    return torch.stack([values(w[e].T).T if trans else values(w[e]) for e in range(E)])
