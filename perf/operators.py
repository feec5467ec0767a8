"""The mixed-precision linear-layer operators and what they are measured on.

Four operators: the matrix product with bias, activation and residual in its epilogue
(``forward``), its gradient (``grad``), the global norm of a list of gradients (``norm``) and
the clipping of such a list to a norm (``clip``). Matrices are column-major as everywhere in
the library: a matrix with leading dimension ``ld`` is held in a torch tensor of shape
``[columns, ld]`` whose first ``rows`` entries of each row are the column.

``run`` computes the plain form in 32 bits (elementary torch operations), or, where ``own``
is true, calls the library. ``exact`` computes the same from the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def listed():
    return [
        # one token through a small projection of a served model: launch latency counts
        dict(name="forward_token_small", op="forward", dtype="fp16", ta="T", tb="N", M=1024, N=1, K=1024,
             act="none", bias=True, residual=True, pre=False, alpha=1.0, beta=1.0, pad=8),
        # one token through a wide up-projection: the weights stream from HBM
        dict(name="forward_token_wide", op="forward", dtype="bf16", ta="T", tb="N", M=16384, N=1, K=4096,
             act="silu", bias=False, residual=False, pre=False, alpha=1.0, beta=0.0, pad=8),
        # a decoding batch of odd size through a down-projection with its residual
        dict(name="forward_batch_37", op="forward", dtype="bf16", ta="T", tb="N", M=4096, N=37, K=10240,
             act="none", bias=True, residual=True, pre=False, alpha=1.0, beta=1.0, pad=8),
        # a ragged prompt, odd sizes everywhere and leading dimensions that equal the odd row counts
        dict(name="forward_ragged", op="forward", dtype="bf16", ta="T", tb="N", M=5003, N=1237, K=1365,
             act="gelu", bias=True, residual=False, pre=False, alpha=1.0, beta=0.0, pad=1),
        # training: the up-projection of a transformer block, pre-activation kept for the gradient
        dict(name="forward_train", op="forward", dtype="bf16", ta="T", tb="N", M=16384, N=8192, K=4096,
             act="gelu_tanh", bias=True, residual=False, pre=True, alpha=1.0, beta=0.0, pad=8),
        # a short fine-tuning batch, a small layer
        dict(name="grad_small", op="grad", dtype="fp16", ta="T", tb="N", M=1024, N=256, K=768,
             act="silu", bias=True, alpha=1.0, pad=8),
        # a ragged batch, weights stored untransposed
        dict(name="grad_ragged", op="grad", dtype="bf16", ta="N", tb="N", M=2999, N=1777, K=2048,
             act="relu", bias=True, alpha=0.5, pad=8),
        # training: the gradient of an up-projection
        dict(name="grad_train", op="grad", dtype="bf16", ta="T", tb="N", M=16384, N=8192, K=4096,
             act="gelu_tanh", bias=True, alpha=1.0, pad=8),
        # the gradients of a small adapter, in 32 bits
        dict(name="norm_small", op="norm", dtype="fp32", tensors=24, elements=600_000, odd=True, clip=0.0, out="fp32"),
        # the gradients of a model of a billion parameters
        dict(name="norm_large", op="norm", dtype="bf16", tensors=290, elements=1_000_000_000, odd=False, clip=0.0,
             out="bf16"),
        # a small adapter's gradients, clipped
        dict(name="clip_small", op="clip", dtype="bf16", tensors=64, elements=4_000_000, odd=True, clip=0.25, out="fp32"),
        # a model's gradients, clipped
        dict(name="clip_large", op="clip", dtype="bf16", tensors=290, elements=700_000_000, odd=False, clip=0.25,
             out="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; half of them odd, the others a multiple of 8 where one fits."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v | 1 if rng.random() < 0.5 else max(v // 8 * 8, min(lo, 8))


def draw(rng: random.Random):
    kind = rng.choice(("forward", "forward", "grad", "norm", "clip"))
    if kind in ("forward", "grad"):
        while True:
            M, K = _log(rng, 64, 16384), _log(rng, 64, 16384)
            N = _log(rng, 1, 8192) if kind == "forward" else _log(rng, 16, 8192)
            if M * N * K <= 2 ** 39:
                break
        case = dict(op=kind, dtype=rng.choice(("bf16", "bf16", "fp16")), ta=rng.choice("TTN"), tb=rng.choice("NNT"),
                    M=M, N=N, K=K, act=rng.choice(ACTS), bias=rng.random() < 0.7,
                    alpha=rng.choice((1.0, 1.0, 0.5)), pad=rng.choice((1, 8, 8)))
        if kind == "forward":
            residual = rng.random() < 0.5
            case.update(residual=residual, beta=rng.choice((1.0, 0.5)) if residual else 0.0, pre=rng.random() < 0.4)
        return case
    tensors = rng.randint(1, 400)
    return dict(op=kind, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), tensors=tensors,
                elements=max(tensors, _log(rng, 20_000, 400_000_000)), odd=rng.random() < 0.5,
                clip=rng.choice((0.1, 0.5, 2.0)) if kind == "clip" else 0.0,
                out=rng.choice(("fp32", "fp16", "bf16")) if kind == "clip" else "fp32")


# ------------------------------------------------------------------ inputs
def _ld(rows, pad):
    return -(-rows // pad) * pad


def _matrix(gen, rows, cols, dtype, pad, scale):
    """A column-major rows x cols matrix: the tensor [cols, ld] that holds it."""
    t = torch.empty(cols, _ld(rows, pad), dtype=torch.float32, device="cuda")
    t.normal_(0.0, scale, generator=gen)
    return t.to(dtype)


def _sizes(case):
    """Element counts of the list: matrices of a few sizes and, one in three, a vector beside them."""
    rng = random.Random(case["tensors"] * 1000003 + case["elements"])
    weights = [rng.choice((1.0, 1.0, 3.0)) if i % 3 else 0.001 for i in range(case["tensors"])]
    total = sum(weights)
    sizes = [max(1, int(case["elements"] * w / total)) for w in weights]
    return [n | 1 if case["odd"] else max(8, n // 8 * 8) for n in sizes]


def _packed(sizes, dtype):
    """One buffer, as a training loop keeps its gradients, and a view of it for each tensor, one behind the other."""
    flat = torch.zeros(sum(sizes), dtype=dtype, device="cuda")
    return flat, list(flat.split(sizes))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": dict(case)}
    dt = DTYPES[case["dtype"]]
    if case["op"] in ("forward", "grad"):
        M, N, K, pad = case["M"], case["N"], case["K"], case["pad"]
        a_rows, a_cols = (M, K) if case["ta"] == "N" else (K, M)
        b_rows, b_cols = (K, N) if case["tb"] == "N" else (N, K)
        # weights of a trained layer have entries of about 1/sqrt(K), activations of about 1
        s["A"] = _matrix(gen, a_rows, a_cols, dt, pad, K ** -0.5)
        s["B"] = _matrix(gen, b_rows, b_cols, dt, pad, 1.0)
        s["bias"] = torch.empty(M, device="cuda").normal_(0.0, 0.2, generator=gen).to(dt) if case["bias"] else None
        if case["op"] == "forward":
            s["C"] = _matrix(gen, M, N, dt, pad, 1.0) if case["residual"] else None
            s["D"] = torch.zeros(N, _ld(M, pad), dtype=dt, device="cuda")
            s["P"] = torch.zeros(N, _ld(M, pad), dtype=dt, device="cuda") if case["pre"] else None
        else:
            s["pre"] = _matrix(gen, M, N, dt, pad, 1.0)
            # a loss that is a mean over tokens: its gradients are small, and still far from the types' borders
            s["dD"] = _matrix(gen, M, N, dt, pad, 0.05)
            s["dA"] = torch.zeros_like(s["A"])
            s["dB"] = torch.zeros_like(s["B"])
            s["dbias"] = torch.zeros(M, dtype=dt, device="cuda") if case["bias"] else None
        return s
    sizes = _sizes(case)
    # gradients of different layers differ in size by an order of magnitude or so
    scales = torch.empty(len(sizes), device="cuda").uniform_(-1.0, 0.5, generator=gen)
    s["grads"] = _packed(sizes, dt)[1]
    for i, n in enumerate(sizes):
        s["grads"][i].copy_(torch.empty(n, device="cuda").normal_(0.0, 1.0, generator=gen) * (1e-3 * 10.0 ** scales[i]))
    if case["op"] == "clip":
        s["out_flat"], s["out"] = _packed(sizes, DTYPES[case["out"]])
        s["max_norm"] = float(case["clip"])
    s["norm"] = torch.zeros(1, dtype=torch.float32, device="cuda")
    return s


# ------------------------------------------------------------------ the plain form
def _op(t, rows, trans):
    """op(X) in 32 bits of the column-major matrix that `t` holds."""
    x = t[:, :rows].float()
    return x if trans == "T" else x.T


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * (1.0 / math.sqrt(2.0))))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * (1.0 / math.sqrt(2.0)))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if act == "silu":
        g = 1.0 / (1.0 + torch.exp(-z))
        return g * (1.0 + z * (1.0 - g))
    return torch.ones_like(z)


def _plain_forward(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    M, N, K = c["M"], c["N"], c["K"]
    z = _op(s["A"], M if c["ta"] == "N" else K, c["ta"]) @ _op(s["B"], K if c["tb"] == "N" else N, c["tb"])
    z = z * c["alpha"]
    if s["bias"] is not None:
        z = z + s["bias"].float()[:, None]
    d = _act(z, c["act"])
    if s["C"] is not None:
        d = d + c["beta"] * s["C"][:, :M].float().T
    out = {"D": d.T.to(dt)}
    if c["pre"]:
        out["pre"] = z.T.to(dt)
    return out


def _plain_grad(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    M, N, K = c["M"], c["N"], c["K"]
    a = _op(s["A"], M if c["ta"] == "N" else K, c["ta"])
    b = _op(s["B"], K if c["tb"] == "N" else N, c["tb"])
    dz = s["dD"][:, :M].float().T * _act_grad(s["pre"][:, :M].float().T, c["act"])
    da = c["alpha"] * (dz @ b.T)
    db = c["alpha"] * (a.T @ dz)
    # back to the layout in which the gradients lie: [columns, rows]
    out = {"dA": (da.T if c["ta"] == "N" else da).to(dt), "dB": (db.T if c["tb"] == "N" else db).to(dt)}
    if s["dbias"] is not None:
        out["dbias"] = dz.sum(dim=1).to(dt)
    return out


def _plain_norm(s):
    # squares are summed in 64 bits: the sums are long
    total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum()
    return total.sqrt()


def _plain_clip(s):
    norm = _plain_norm(s)
    scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, torch.ones_like(norm)).float()
    for g, o in zip(s["grads"], s["out"]):
        o.copy_(g.float() * scale)
    return {"norm": norm.float().reshape(1), "out": s["out_flat"]}


# ------------------------------------------------------------------ the library
def _library():
    import __graft_entry__
    pl = __graft_entry__.load_package()
    pl.lib()
    return pl


def _own_forward(s):
    pl, c = _library(), s["case"]
    dt = DTYPES[c["dtype"]]
    ty, act = (pl.BF16 if dt == torch.bfloat16 else pl.F16), ACTS.index(c["act"])
    A, B, D, P = s["A"], s["B"], s["D"], s["P"]
    M, N, K = c["M"], c["N"], c["K"]
    if "scratch" not in s:
        n = pl.tile_gemm_act_scratch_bytes(ty, c["ta"], c["tb"], M, N, K, A, A.shape[1], B, B.shape[1])
        s["scratch"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        s["scratch_bytes"] = n
    pl.tile_gemm_act(0, ty, c["ta"], c["tb"], M, N, K, c["alpha"], A, A.shape[1], B, B.shape[1], c["beta"], s["C"],
                     D.shape[1], D, D.shape[1], bias=s["bias"], act=act, pre=P, ldPre=D.shape[1],
                     scratch=s["scratch"], scratch_bytes=s["scratch_bytes"],
                     stream=torch.cuda.current_stream().cuda_stream)
    out = {"D": D[:, :M]}
    if c["pre"]:
        out["pre"] = P[:, :M]
    return out


def _own_grad(s):
    pl, c = _library(), s["case"]
    dt = DTYPES[c["dtype"]]
    ty, act = (pl.BF16 if dt == torch.bfloat16 else pl.F16), ACTS.index(c["act"])
    A, B, pre, dD, dA, dB = s["A"], s["B"], s["pre"], s["dD"], s["dA"], s["dB"]
    M, N, K = c["M"], c["N"], c["K"]
    if "scratch" not in s:
        n = pl.tile_gemm_act_grad_scratch_bytes(ty, c["ta"], c["tb"], M, N, K, A, A.shape[1], B, B.shape[1], act)
        s["scratch"] = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        s["scratch_bytes"] = n
    pl.tile_gemm_act_grad(0, ty, c["ta"], c["tb"], M, N, K, c["alpha"], A, A.shape[1], B, B.shape[1], act, pre,
                          pre.shape[1], dD, dD.shape[1], dA=dA, lddA=dA.shape[1], dB=dB, lddB=dB.shape[1],
                          dbias=s["dbias"], scratch=s["scratch"], scratch_bytes=s["scratch_bytes"],
                          stream=torch.cuda.current_stream().cuda_stream)
    out = {"dA": dA[:, :M if c["ta"] == "N" else K], "dB": dB[:, :K if c["tb"] == "N" else N]}
    if s["dbias"] is not None:
        out["dbias"] = s["dbias"]
    return out


def _own_list(s):
    """The list of gradients, described once and kept, as a training loop keeps it, and its scratch."""
    pl = _library()
    if "list" not in s:
        s["list"] = pl.TensorList(s["grads"], s.get("out"))
        s["scratch"] = torch.empty(pl.tile_grad_norm_scratch_bytes(s["list"]), dtype=torch.uint8, device="cuda")
    return pl, s["list"], s["scratch"]


def _own_norm(s):
    pl, grads, scratch = _own_list(s)
    pl.tile_grad_norm(0, grads, scratch, norm=s["norm"], stream=torch.cuda.current_stream().cuda_stream)
    return s["norm"]


def _own_clip(s):
    pl, grads, scratch = _own_list(s)
    pl.tile_grad_clip(0, grads, s["max_norm"], scratch, norm=s["norm"], stream=torch.cuda.current_stream().cuda_stream)
    return {"norm": s["norm"], "out": s["out_flat"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"forward": _own_forward, "grad": _own_grad, "norm": _own_norm, "clip": _own_clip}[op](state)
    if op == "forward":
        return _plain_forward(state)
    if op == "grad":
        return _plain_grad(state)
    if op == "norm":
        return _plain_norm(state).float().reshape(1)
    return _plain_clip(state)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("forward", "grad"):
        M, N, K = case["M"], case["N"], case["K"]
        if case["op"] == "forward":
            values = M * K + K * N + M * N * (1 + bool(case["residual"]) + bool(case["pre"])) + M * bool(case["bias"])
            return {"bytes": e * values, "flops": 2.0 * M * N * K}
        # operands in, their gradients out; the incoming gradient, and the pre-activation where it is looked at
        values = 2 * (M * K + K * N) + M * N * (1 + (case["act"] != "none")) + M * bool(case["bias"])
        return {"bytes": e * values, "flops": 4.0 * M * N * K}
    n = sum(_sizes(case))
    if case["op"] == "norm":
        return {"bytes": e * n, "flops": 2.0 * n}
    return {"bytes": n * (e + (4 if case["out"] == "fp32" else 2)), "flops": 3.0 * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_act(z, act):
    """(act(z), act'(z))"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0.0), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device=z.device))
    if act == "silu":
        g = torch.sigmoid(z)
        return z * g, g + z * g * (1 - g)
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / 2 ** 0.5)
        return z * cdf, cdf + z * torch.exp(-z ** 2 / 2) / (2 * math.pi) ** 0.5
    u = (2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)
    g = torch.sigmoid(2 * u)                    # (1 + tanh(u)) / 2
    return z * g, g + z * 2 * g * (1 - g) * (2 / math.pi) ** 0.5 * (1 + 3 * 0.044715 * z ** 2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "clip"):
        norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["grads"]))
        if case["op"] == "norm":
            return torch.tensor([norm], dtype=torch.float64)
        k = s["max_norm"] / norm if norm > s["max_norm"] else 1.0
        return {"norm": torch.tensor([norm], dtype=torch.float64), "out": torch.cat([g.double() * k for g in s["grads"]])}
    M, N, K = case["M"], case["N"], case["K"]
    # in the layout of the storage: xt[j, i] is entry (i, j), so a product of matrices turns round
    a = s["A"].double()[:, :M] if case["ta"] == "N" else s["A"].double()[:, :K].t()      # [K, M]
    b = s["B"].double()[:, :K] if case["tb"] == "N" else s["B"].double()[:, :N].t()      # [N, K]
    if case["op"] == "forward":
        z = torch.matmul(b, a).mul_(case["alpha"])                                       # [N, M]
        if s["bias"] is not None:
            z += s["bias"].double()
        d = _exact_act(z, case["act"])[0]
        if s["C"] is not None:
            d = d + s["C"].double()[:, :M] * case["beta"]
        return {"D": d, "pre": z} if case["pre"] else {"D": d}
    dz = _exact_act(s["pre"].double()[:, :M], case["act"])[1].mul_(s["dD"].double()[:, :M])   # [N, M]
    da = torch.matmul(b.t(), dz).mul_(case["alpha"])                                     # [K, M]
    db = torch.matmul(dz, a.t()).mul_(case["alpha"])                                     # [N, K]
    out = {"dA": da if case["ta"] == "N" else da.t(), "dB": db if case["tb"] == "N" else db.t()}
    if s["dbias"] is not None:
        out["dbias"] = dz.sum(0)
    return out
