"""Tables behind the choices of the adapter calls (`gemm_lora`, `gemm_lora_backward`), on one GPU.

    python cute-examples_b200/tests/lora_bench.py [--few] [--wave] [--ring] [--plan] [--low]      (all without a flag)

  --few   up to 128 rows and a long K: tiles of 256 against 128 columns, cut in four, and which the library takes
  --wave  129 to 1024 rows, output of less than a wave: the shared planner's tiles against the library's choice
  --ring  the low-rank rows through the short against the deep ring, and which the library takes
  --plan  LoraPlan.update by rows and adapters
  --low   the low-rank rows alone (gemm_sm100_lora_low)

Times are microseconds per call from CUDA graphs of six calls over rotating operands (sets of more than 300 MB where that fits
into six), the best of several replays, the variants in alternation.  Forward calls stand behind a 2048 x 2048 x 2048 GEMM ("behind") or
follow one another ("alone"); gradients are part of a step of a forward and a backward call.  Adapters: `one` / `runs` (one
stretch of rows each) / `mixed` (row m uses adapter m mod adapters).  The reference has no counterpart.
"""
import argparse
import ctypes
import os
import sys

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

import torch  # noqa: E402

import gemm_kernels as gk  # noqa: E402

DTYPE = torch.bfloat16


def rnd(*shape):
    return torch.randn(*shape, device="cuda").to(DTYPE)


def graph_us(fn, calls=6, replays=5):
    for i in range(3):
        fn(i)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(calls):
            fn(i)
    graph.replay()
    torch.cuda.synchronize()
    best = 1e9
    for _ in range(replays):
        a, b = torch.cuda.Event(True), torch.cuda.Event(True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / calls * 1e3)
    return best


def adapters_of(M, G, kind):
    rows = torch.arange(M, device="cuda")
    return (rows * G // M if kind != "mixed" else rows % G).to(torch.int32)


class Shape:
    """Operands of one shape in rotating sets, and the calls that are timed."""

    front = None
    options = {}                                           # set around the adapter calls only

    def __init__(self, M, N, K, G, R, kind, gradient=False):
        each = 2 * (N * K + M * K + M * N * (2 if gradient else 1) + G * R * (N + K))
        self.sets = [(rnd(M, K), rnd(N, K), rnd(G, R, K), rnd(G, N, R), rnd(M, N) if gradient else None)
                     for _ in range(max(2, min(6, int(3e8 // each))))]
        self.plan = gk.LoraPlan(adapters_of(M, G, kind), G)
        self.out, self.low = torch.empty(M, N, dtype=DTYPE, device="cuda"), torch.empty(M, R, dtype=DTYPE, device="cuda")
        if Shape.front is None:
            Shape.front = (rnd(2048, 2048), rnd(2048, 2048), torch.empty(2048, 2048, dtype=DTYPE, device="cuda"))

    def alone(self, i, gradient=False):
        A, B, down, up, dC = self.sets[i % len(self.sets)]
        for name, value in self.options.items():
            gk.set_option(name, value)
        gk.gemm_lora(A, B, down, up, self.plan, out=self.out, low=self.low)
        if gradient:
            gk.gemm_lora_backward(dC, A, B, down, up, self.plan, low=self.low)
        for name in self.options:
            gk.set_option(name, 0 if name == "max_ctas" else -1)

    def behind(self, i):
        gk.gemm_tn(Shape.front[0], Shape.front[1], out=Shape.front[2])
        self.alone(i)

    def step(self, i):
        self.alone(i, gradient=True)

    def compare(self, fn, settings):
        """Best time under each of the option settings, in alternation."""
        best = [1e9] * len(settings)
        for _ in range(3):
            for i, self.options in enumerate(settings):
                best[i] = min(best[i], graph_us(fn))
        return best


def change(a, b):
    return f"{a:6.1f} -> {b:6.1f} ({100 * (b / a - 1):+5.1f} %)"


def few():
    cut = {"split_k": 4, "sk_cluster": 1}
    print("up to 128 rows, cut in four: 256 -> 128 columns, the library's choice")
    for M in (16, 128):
        for N in (1024, 2560, 3200, 3584, 3712, 3968, 4224):
            for K in (8704, 14336):
                for G, R in ((1, 16), (8, 64), (16, 64), (28, 64), (64, 64)):
                    if G > M:
                        continue
                    s = Shape(M, N, K, G, R, "mixed")
                    chosen = gk.describe_lora_plan(M, N, K, R, G).split("tile=128x")[1].split("x")[0]
                    pairs = [s.compare(f, [{"tile_config": 2, **cut}, {"tile_config": 12, **cut}]) for f in (s.behind, s.alone)]
                    print(f"{M:4d} x {N} x {K:5d} {G:2d} adapters of rank {R}: behind {change(*pairs[0])}  alone {change(*pairs[1])}  takes {chosen}",
                          flush=True)


def wave():
    print("outputs of less than a wave: the planner's tiles -> the library's choice")
    sizes = [(False, m, n, k) for m, n in ((512, 4352), (1024, 2048), (1024, 2304), (256, 9216)) for k in (512, 1024, 2048)]
    sizes += [(False, m, n, k) for m, n in ((256, 4608), (512, 2304), (512, 1024), (256, 2048), (1024, 512), (256, 2560)) for k in (4096, 8192)]
    sizes += [(True, m, n, k) for m, k in ((256, 8704), (512, 4352), (512, 4096), (1024, 2048), (700, 2688)) for n in (1024, 2560, 4096)]
    sizes += [(True, m, n, k) for m, k in ((1024, 1024), (512, 1792), (256, 4096)) for n in (4096, 5120)]
    sizes += [(True, m, n, k) for m, k in ((1024, 512), (512, 1024), (512, 1280)) for n in (8192, 14336)]
    for gradient, M, N, K in sizes:
        line = []
        for G, R, kind in ((1, 64, "one"), (4, 32, "runs"), (16, 16, "mixed")):
            s = Shape(M, N, K, G, R, kind, gradient)
            if gk.describe_lora_plan(M, N, K, R, G, gradient=gradient).startswith("planner"):
                line.append("planner's")
                continue
            line.append(change(*s.compare(s.step if gradient else s.behind, [{"max_ctas": gk.num_sms()}, {"max_ctas": 0}])))
        print(f"{'dA ' if gradient else 'C  '}{M:4d} x {K if gradient else N} x {N if gradient else K}: " + "  ".join(line), flush=True)


def ring():
    print("low-rank rows: short -> deep ring, the library's choice")
    for M, G, R, kind in ((16, 8, 64, "mixed"), (64, 16, 64, "mixed"), (64, 32, 64, "mixed"), (128, 64, 16, "mixed"), (512, 1, 64, "one"),
                          (700, 1, 64, "one"), (1100, 1, 64, "one"), (1100, 8, 64, "mixed")):
        for N, K in ((1024, 8192), (4096, 4096), (4096, 14336), (8192, 8192)):
            s = Shape(M, N, K, G, R, kind)
            chosen = gk.describe_lora_plan(M, N, K, R, G).split(", ")[-1]
            pairs = [s.compare(f, [{"lora_ring": 0}, {"lora_ring": 1}]) for f in (s.behind, s.alone)]
            print(f"{M:4d} x {N} x {K:5d} {G:2d} adapters of rank {R} {kind:5s}: behind {change(*pairs[0])}  alone {change(*pairs[1])}  takes the {chosen}",
                  flush=True)


def plan():
    counts = (1, 16, 64, 512, 4096)
    print("LoraPlan.update, int32 / int64 indices, adapters: " + ", ".join(map(str, counts)))
    for M in (1, 64, 128, 1024, 8192, 65536):
        line = []
        for G in counts:
            ids = torch.randint(-1, G, (M,), device="cuda", dtype=torch.int32)
            wide = ids.long()
            p = gk.LoraPlan(ids, G)
            calls = 30 if M * G < 1e8 else 4
            line.append(f"{graph_us(lambda i: p.update(ids), calls):.1f} / {graph_us(lambda i: p.update(wide), calls):.1f}")
        print(f"{M:6d} rows: " + "  ".join(line), flush=True)


class LoraArgs(ctypes.Structure):
    I, L, P = ctypes.c_int, ctypes.c_long, ctypes.c_void_p
    _fields_ = [("M", I), ("N", I), ("K", I), ("R", I), ("adapters", I), ("dtype", I), ("A", P), ("B", P), ("down", P), ("up", P), ("lda", L),
                ("ldb", L), ("ld_down", L), ("stride_down", L), ("ld_up", L), ("stride_up", L), ("scales", P), ("scale", ctypes.c_float), ("plan", P)]


def low():
    call = ctypes.CDLL(gk.LIBRARY_PATH).gemm_sm100_lora_low
    call.argtypes = [ctypes.POINTER(LoraArgs), ctypes.c_void_p, ctypes.c_long, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int)]
    print("low-rank rows alone")
    for M, K, G, R, kind in ((8192, 4096, 1, 16, "one"), (8192, 14336, 4, 64, "runs"), (64, 14336, 32, 64, "mixed"), (128, 4096, 64, 16, "mixed"),
                             (2048, 4096, 8, 32, "runs"), (2048, 4096, 16, 32, "mixed"), (1, 4096, 4, 16, "one")):
        s = Shape(M, 8, K, G, R, kind)

        def run(i):
            A, _, down, _, _ = s.sets[i % len(s.sets)]
            a = LoraArgs(M=M, N=8, K=K, R=R, adapters=G, dtype=0, A=A.data_ptr(), down=down.data_ptr(), lda=K, ld_down=K, stride_down=R * K,
                         scale=1.0, plan=s.plan.buffer.data_ptr())
            assert call(ctypes.byref(a), s.low.data_ptr(), R, torch.cuda.current_stream().cuda_stream, None) == 0

        us = graph_us(run)
        read = 2 * (M * K + min(G, M) * R * K)
        print(f"{M:5d} x {K} {G:2d} adapters of rank {R} {kind:5s}: {us:6.1f} us, {read / us / 1e6:.2f} TB/s", flush=True)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parts = {"few": few, "wave": wave, "ring": ring, "plan": plan, "low": low}
    for name in parts:
        ap.add_argument("--" + name, action="store_true")
    args = ap.parse_args()
    wanted = [name for name in parts if getattr(args, name)] or list(parts)
    with torch.no_grad():
        for name in wanted:
            parts[name]()
