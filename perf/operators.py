"""What is measured of the low-rank adapter operators: the cases, their inputs and the calls.

C = A B^T + s_g (A down_g^T) up_g^T for every row of A, where g is the adapter of that row: a projection that
many requests share, each with a low-rank adapter of its own (or none), and its gradients.

  "forward"   gemm_lora                       one projection of a serving batch
  "backward"  gemm_lora_backward              gradients of A and of the adapters, the low-rank rows recomputed
  "train"     gemm_lora, gemm_lora_backward   a training step's share of one projection; the low-rank rows are kept

With `own` false the same results come from elementary torch operations in 32 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def _case(name, op, rows, n, k, rank, adapters, requests, order, bare, dtype):
    return {"name": name, "op": op, "rows": rows, "n": n, "k": k, "rank": rank, "adapters": adapters,
            "requests": requests, "order": order, "bare": bare, "dtype": dtype}


def listed():
    return [
        # one token of one request: pure latency, W is all that moves
        _case("decode_1x4096x4096_r16", "forward", 1, 4096, 4096, 16, 4, 1, "requests", False, "bf16"),
        # a small decode batch on the widest projection, every request with an adapter of its own
        _case("decode_16x28672x8192_r16", "forward", 16, 28672, 8192, 16, 16, 16, "requests", False, "bf16"),
        # a decode batch over many adapters of a higher rank, down-projection, some requests without one
        _case("decode_64x4096x14336_r64_fp16", "forward", 64, 4096, 14336, 64, 32, 64, "requests", True, "fp16"),
        # a full decode batch, up-projection, adapters shared by two requests each
        _case("decode_128x14336x4096_r16", "forward", 128, 14336, 4096, 16, 64, 128, "requests", True, "bf16"),
        # sizes that fit no tile: ragged rows and columns, the smallest rank
        _case("odd_77x1000x1032_r8_fp16", "forward", 77, 1000, 1032, 8, 5, 9, "requests", True, "fp16"),
        # prompts of several requests beside one another
        _case("prefill_2048x4096x4096_r32", "forward", 2048, 4096, 4096, 32, 8, 11, "requests", True, "bf16"),
        # a large prompt batch on the up-projection
        _case("prefill_8192x14336x4096_r64", "forward", 8192, 14336, 4096, 64, 4, 6, "requests", False, "bf16"),
        # fine-tuning of one adapter
        _case("backward_8192x4096x4096_r16", "backward", 8192, 4096, 4096, 16, 1, 1, "requests", False, "bf16"),
        # rows of many adapters in no order
        _case("backward_2048x4096x4096_r32_shuffled", "backward", 2048, 4096, 4096, 32, 16, 24, "shuffled", True, "bf16"),
        # a short ragged batch in the other type
        _case("backward_300x1000x520_r8_fp16", "backward", 300, 1000, 520, 8, 3, 5, "requests", True, "fp16"),
        # a step over adapters of several tasks, forward and backward together
        _case("train_1024x8192x1024_r128", "train", 1024, 8192, 1024, 128, 2, 3, "requests", False, "bf16"),
        _case("train_8192x14336x4096_r64", "train", 8192, 14336, 4096, 64, 8, 10, "requests", True, "bf16"),
    ]


def draw(rng):
    """One more case: sizes over the logarithm of their ranges, products of sizes bounded by the largest listed case."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["forward", "forward", "backward", "train"])
    while True:
        rows = log_int(1, 8192) if op == "forward" else log_int(64, 8192)
        n, k = log_int(32, 3584) * 8, log_int(32, 1792) * 8
        if rows * n * k <= 8192 * 14336 * 4096 and n * k <= 28672 * 8192:
            break
    rank = 8 * log_int(1, 16)
    adapters = log_int(1, 64)
    requests = rows if op == "forward" and rows <= 128 and rng.random() < 0.7 else min(rows, log_int(1, 96))
    order = "shuffled" if rng.random() < 0.25 else "requests"
    return {"op": op, "rows": rows, "n": n, "k": k, "rank": rank, "adapters": adapters, "requests": requests,
            "order": order, "bare": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "fp16"])}


def _requests(case):
    """Adapter slot of every request (-1: none); the seed decides which adapter a slot is."""
    return [-1 if case["bare"] and i % 8 == 7 else i % case["adapters"] for i in range(case["requests"])]


def _adapter_ids(case, seed):
    rng = np.random.default_rng(seed)
    slots = np.array(_requests(case), dtype=np.int64)
    names = rng.permutation(case["adapters"])
    of_request = np.where(slots >= 0, names[np.maximum(slots, 0)], -1)
    count, rows = len(slots), case["rows"]
    # ragged requests: every one has a row, the others fall by exponential weights
    weights = rng.exponential(size=count)
    lengths = 1 + rng.multinomial(rows - count, weights / weights.sum())
    ids = np.repeat(of_request, lengths)
    if case["order"] == "shuffled":
        rng.shuffle(ids)
    return ids.astype(np.int32)


def _inputs(case, seed):
    dtype = DTYPES[case["dtype"]]
    rows, n, k, rank, adapters = (case[x] for x in ("rows", "n", "k", "rank", "adapters"))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(shape, std):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    s = {"A": normal((rows, k), 1.0), "B": normal((n, k), k ** -0.5),
         "down": normal((adapters, rank, k), k ** -0.5), "up": normal((adapters, n, rank), 0.25 * rank ** -0.5)}
    s["scale"] = 0.5 + 1.5 * torch.rand((adapters,), generator=gen, device="cuda")
    if case["op"] != "forward":
        s["dC"] = normal((rows, n), 0.5)
    ids = _adapter_ids(case, seed)
    s["ids"] = torch.from_numpy(ids).cuda()
    return s, ids


def prepare(case, seed):
    s, ids = _inputs(case, seed)
    s["op"] = case["op"]
    if own:
        package = os.path.join(os.getcwd(), "cute-examples_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import gemm_kernels

        s["gk"] = gemm_kernels
        s["plan"] = gemm_kernels.LoraPlan(s["ids"], case["adapters"])
    else:
        s["rows_of"] = [(int(g), torch.from_numpy(np.flatnonzero(ids == g)).cuda()) for g in np.unique(ids) if g >= 0]
    return s


def _run_own(s):
    gk, plan = s["gk"], s["plan"]
    if s["op"] == "forward":
        return gk.gemm_lora(s["A"], s["B"], s["down"], s["up"], plan, scale=s["scale"])
    if s["op"] == "backward":
        return gk.gemm_lora_backward(s["dC"], s["A"], s["B"], s["down"], s["up"], plan, scale=s["scale"])
    low = torch.empty((s["A"].shape[0], s["down"].shape[1]), dtype=s["A"].dtype, device=s["A"].device)
    C = gk.gemm_lora(s["A"], s["B"], s["down"], s["up"], plan, scale=s["scale"], low=low)
    grads = gk.gemm_lora_backward(s["dC"], s["A"], s["B"], s["down"], s["up"], plan, scale=s["scale"], low=low)
    return (C, low) + tuple(grads)


def run(state):
    if own:
        return _run_own(state)
    s = state
    dtype = s["A"].dtype
    A, B = s["A"].float(), s["B"].float()
    low = torch.zeros((A.shape[0], s["down"].shape[1]), device=A.device)
    for g, rows in s["rows_of"]:
        low[rows] = (A[rows] @ s["down"][g].float().T) * s["scale"][g]
    out = ()
    if s["op"] != "backward":
        C = A @ B.T
        for g, rows in s["rows_of"]:
            C[rows] += low[rows] @ s["up"][g].float().T
        if s["op"] == "forward":
            return C.to(dtype)
        out = (C.to(dtype), low.to(dtype))
        del C
    dC = s["dC"].float()
    dA = dC @ B
    d_down = torch.zeros_like(s["down"], dtype=torch.float32)
    d_up = torch.zeros_like(s["up"], dtype=torch.float32)
    for g, rows in s["rows_of"]:
        dC_g = dC[rows]
        d_low = (dC_g @ s["up"][g].float()) * s["scale"][g]
        dA[rows] += d_low @ s["down"][g].float()
        d_down[g] = d_low.T @ A[rows]
        d_up[g] = dC_g.T @ low[rows]
    return out + (dA.to(dtype), d_down.to(dtype), d_up.to(dtype))


def exact(case, seed):
    """From the definition with the adapters merged into the weights: rows of adapter g see W_g = B + s_g up_g down_g,
    dA = dC W_g, and with D = dC_g^T A_g the gradient of W_g: d_down = s_g up_g^T D, d_up = s_g D down_g^T."""
    s, ids = _inputs(case, seed)
    rows, n = case["rows"], case["n"]
    weight = s["B"].double()
    forward, backward = case["op"] != "backward", case["op"] != "forward"
    C = torch.zeros((rows, n), dtype=torch.float64, device="cuda") if forward else None
    low = torch.zeros((rows, case["rank"]), dtype=torch.float64, device="cuda")
    if backward:
        dA = torch.zeros((rows, case["k"]), dtype=torch.float64, device="cuda")
        d_down = torch.zeros_like(s["down"], dtype=torch.float64)
        d_up = torch.zeros_like(s["up"], dtype=torch.float64)
    for g in np.unique(ids):
        at = torch.from_numpy(np.flatnonzero(ids == g)).cuda()
        x = s["A"][at].double()
        merged = weight
        if g >= 0:
            scale = s["scale"][g].double()
            down, up = s["down"][g].double(), s["up"][g].double()
            merged = torch.addmm(weight, up * scale, down)
            low[at] = (x * scale) @ down.T
        if forward:
            C[at] = x @ merged.T
        if backward:
            dy = s["dC"][at].double()
            dA[at] = dy @ merged
            if g >= 0:
                d_merged = (dy.T @ x) * scale
                d_down[g] = up.T @ d_merged
                d_up[g] = d_merged @ down.T
    if case["op"] == "forward":
        return C
    grads = (dA, d_down, d_up)
    return grads if case["op"] == "backward" else (C, low) + grads


def work(case):
    rows, n, k, rank, adapters = (case[x] for x in ("rows", "n", "k", "rank", "adapters"))
    requests = _requests(case)
    used = len({g for g in requests if g >= 0})
    adapted = rows * sum(g >= 0 for g in requests) / len(requests)
    weights = n * k + used * rank * (n + k)
    product, thin = 2 * rows * n * k, 2 * adapted * rank
    f_bytes, f_flops = 2 * (rows * k + weights + rows * n) + 4 * rows, product + thin * (n + k)
    # dC, A and the weights in; dA and a gradient for every adapter out
    b_bytes = 2 * (rows * (n + 2 * k) + weights + adapters * rank * (n + k)) + 4 * rows
    b_flops = product + thin * 2 * (n + k)
    if case["op"] == "forward":
        return {"bytes": f_bytes, "flops": f_flops}
    if case["op"] == "backward":
        return {"bytes": b_bytes, "flops": b_flops + thin * k}
    return {"bytes": 2 * (rows * (2 * n + 2 * k + rank) + weights + adapters * rank * (n + k)) + 4 * rows,
            "flops": f_flops + b_flops}
