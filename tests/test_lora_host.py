"""Adapter entry points without a GPU: the C ABI and the binding refuse bad arguments before they touch CUDA."""
import ctypes

import pytest
import torch

from conftest import load_capi

I, L, P, Z, F = ctypes.c_int, ctypes.c_long, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_float


class LoraArgs(ctypes.Structure):
    _fields_ = [("M", I), ("N", I), ("K", I), ("R", I), ("adapters", I), ("dtype", I), ("A", P), ("B", P), ("down", P),
                ("up", P), ("lda", L), ("ldb", L), ("ld_down", L), ("stride_down", L), ("ld_up", L), ("stride_up", L),
                ("scales", P), ("scale", F), ("plan", P)]


def good(**changes):
    """A call that would be accepted; the addresses are never followed because every test breaks something."""
    values = dict(M=32, N=64, K=128, R=16, adapters=4, dtype=0, A=0x1000, B=0x2000, down=0x3000, up=0x4000, lda=128, ldb=128,
                  ld_down=128, stride_down=16 * 128, ld_up=16, stride_up=64 * 16, scales=None, scale=1.0, plan=0x5000)
    values.update(changes)
    return LoraArgs(**values)


@pytest.fixture(scope="module")
def lora():
    lib = load_capi()
    lib.gemm_sm100_lora_plan_bytes.argtypes, lib.gemm_sm100_lora_plan_bytes.restype = [I, I], Z
    lib.gemm_sm100_lora_plan.argtypes = [P, I, I, I, P, Z, P, ctypes.POINTER(I)]
    lib.gemm_sm100_lora_low.argtypes = [ctypes.POINTER(LoraArgs), P, L, P, ctypes.POINTER(I)]
    lib.gemm_sm100_lora.argtypes = [ctypes.POINTER(LoraArgs), P, L, P, L, P, ctypes.POINTER(I)]
    lib.gemm_sm100_lora_backward.argtypes = [ctypes.POINTER(LoraArgs), P, L, P, L, I, P, L, P, L, P, P, P, ctypes.POINTER(I)]
    return lib


NULL, SHAPE, ALIGN, DTYPE, WORKSPACE = 1, 2, 3, 4, 7

COMMON = [
    (dict(M=-1), SHAPE), (dict(N=0), SHAPE), (dict(K=0), SHAPE), (dict(K=124, lda=128), SHAPE), (dict(R=0), SHAPE),
    (dict(R=12), SHAPE), (dict(R=136), SHAPE), (dict(adapters=0), SHAPE), (dict(adapters=4097), SHAPE), (dict(dtype=2), DTYPE),
    (dict(plan=None), NULL),
]
FORWARD = COMMON + [
    (dict(A=None), NULL), (dict(B=None), NULL), (dict(down=None), NULL), (dict(up=None), NULL),
    (dict(A=0x1008), ALIGN), (dict(B=0x2002), ALIGN), (dict(down=0x3004), ALIGN), (dict(up=0x4008), ALIGN),
    (dict(lda=120), SHAPE), (dict(ldb=64), SHAPE), (dict(ld_down=64), SHAPE), (dict(ld_up=8), SHAPE),
    (dict(lda=132), ALIGN), (dict(ld_up=20), ALIGN), (dict(stride_down=16 * 128 - 8), SHAPE), (dict(stride_up=0), SHAPE),
    (dict(stride_down=16 * 128 + 4), ALIGN), (dict(stride_up=64 * 16 + 2), ALIGN),
]


@pytest.mark.parametrize("changes,want", FORWARD)
def test_forward_refuses(lora, changes, want):
    err = I(-7)
    assert lora.gemm_sm100_lora(ctypes.byref(good(**changes)), 0x6000, 64, 0x7000, 16, None, ctypes.byref(err)) == want
    assert err.value == 0


@pytest.mark.parametrize("C,ldc,low,ld_low,want", [
    (None, 64, 0x7000, 16, NULL), (0x6000, 64, None, 16, NULL), (0x6000, 56, 0x7000, 16, SHAPE), (0x6000, 64, 0x7000, 8, SHAPE),
    (0x6004, 64, 0x7000, 16, ALIGN), (0x6000, 64, 0x7008, 16, ALIGN), (0x6000, 68, 0x7000, 16, ALIGN), (0x6000, 64, 0x7000, 20, ALIGN)])
def test_forward_refuses_outputs(lora, C, ldc, low, ld_low, want):
    err = I(0)
    assert lora.gemm_sm100_lora(ctypes.byref(good()), C, ldc, low, ld_low, None, ctypes.byref(err)) == want


@pytest.mark.parametrize("changes,want", COMMON + [(dict(N=60, stride_up=60 * 16), SHAPE), (dict(up=None), NULL), (dict(B=None), NULL),
                                                   (dict(down=None), NULL), (dict(A=None), NULL)])
def test_backward_refuses(lora, changes, want):
    err = I(-7)
    rc = lora.gemm_sm100_lora_backward(ctypes.byref(good(**changes)), 0x6000, 64, 0x7000, 16, 0, 0x8000, 16, 0x9000, 128, 0xA000,
                                       0xB000, None, ctypes.byref(err))
    assert rc == want and err.value == 0


@pytest.mark.parametrize("dC,ld_dc,low,d_low,dA,ld_da,d_down,d_up,want", [
    (None, 64, 0x7000, 0x8000, 0x9000, 128, 0xA000, 0xB000, NULL), (0x6000, 56, 0x7000, 0x8000, 0x9000, 128, 0xA000, 0xB000, SHAPE),
    (0x6000, 64, None, 0x8000, 0x9000, 128, 0xA000, 0xB000, NULL), (0x6000, 64, 0x7000, None, 0x9000, 128, 0xA000, 0xB000, NULL),
    (0x6000, 64, 0x7000, 0x8000, 0x9000, 120, 0xA000, 0xB000, SHAPE), (0x6000, 64, 0x7000, 0x8000, 0x9000, 128, 0xA004, 0xB000, ALIGN),
    (0x6000, 64, 0x7000, 0x8000, 0x9000, 128, 0xA000, 0xB008, ALIGN), (0x6002, 64, 0x7000, 0x8000, 0x9000, 128, 0xA000, 0xB000, ALIGN)])
def test_backward_refuses_tensors(lora, dC, ld_dc, low, d_low, dA, ld_da, d_down, d_up, want):
    err = I(0)
    assert lora.gemm_sm100_lora_backward(ctypes.byref(good()), dC, ld_dc, low, 16, 0, d_low, 16, dA, ld_da, d_down, d_up, None,
                                         ctypes.byref(err)) == want


def test_calls_with_nothing_to_do(lora):
    err = I(0)
    assert lora.gemm_sm100_lora(ctypes.byref(good(M=0, A=None, plan=None)), None, 64, None, 16, None, ctypes.byref(err)) == 0
    assert lora.gemm_sm100_lora_low(ctypes.byref(good(M=0)), None, 16, None, ctypes.byref(err)) == 0
    assert lora.gemm_sm100_lora_backward(ctypes.byref(good()), None, 64, None, 16, 0, None, 16, None, 128, None, None, None,
                                         ctypes.byref(err)) == 0
    assert lora.gemm_sm100_lora(None, None, 0, None, 0, None, ctypes.byref(err)) == NULL


def test_plan_arguments(lora):
    assert lora.gemm_sm100_lora_plan_bytes(-1, 4) == 0 and lora.gemm_sm100_lora_plan_bytes(4, 0) == 0
    assert lora.gemm_sm100_lora_plan_bytes(4, 4097) == 0
    need = lora.gemm_sm100_lora_plan_bytes(300, 7)
    # two tiles of 256 slots (adapter and mask), two lists of the rows, starts of the adapters
    assert need >= 4 * (2 * 256 * 9 + 2 * 300 + 8) and need % 256 == 0
    err = I(0)
    plan = lambda *a: lora.gemm_sm100_lora_plan(*a, None, ctypes.byref(err))  # noqa: E731
    assert plan(0x1000, 0, 300, 7, 0x2000, need - 1) == WORKSPACE
    assert plan(0x1000, 0, 300, 7, 0x2010, need) == WORKSPACE
    assert plan(0x1002, 0, 300, 7, 0x2000, need) == ALIGN
    assert plan(0x1004, 1, 300, 7, 0x2000, need) == ALIGN
    assert plan(None, 0, 300, 7, 0x2000, need) == NULL and plan(0x1000, 0, 300, 7, None, need) == NULL
    assert plan(0x1000, 0, -1, 7, 0x2000, need) == SHAPE and plan(0x1000, 0, 300, 0, 0x2000, need) == SHAPE


def tensors(M=32, N=64, K=128, R=16, G=4, dt=torch.bfloat16):
    z = lambda *s: torch.zeros(*s, dtype=dt)  # noqa: E731
    return dict(A=z(M, K), B=z(N, K), down=z(G, R, K), up=z(G, N, R), plan=torch.zeros(8, dtype=torch.uint8), plan_rows=M,
                plan_adapters=G, plan_stream=0, scales=None, scale=1.0, out=z(M, N), low=z(M, R))


Z16 = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731


@pytest.mark.parametrize("changes,message", [
    (dict(A=Z16(128)), "2D"), (dict(down=Z16(16, 128)), "3D"), (dict(B=Z16(64, 120)), "Inner dimensions"),
    (dict(B=torch.zeros(64, 128)), "same dtype"), (dict(up=Z16(4, 64, 8)), "up must be of shape"),
    (dict(up=Z16(3, 64, 16)), "up must be of shape"), (dict(down=Z16(4, 16, 120)), "down must be of shape"),
    (dict(plan_rows=31), "31 rows"), (dict(plan_adapters=5), "5 adapters"), (dict(out=Z16(32, 72)), "out must be of shape"),
    (dict(low=Z16(32, 8)), "low must be of shape"), (dict(A=Z16(32, 256)[:, ::2]), "unit stride"),
    (dict(scales=torch.ones(3)), "scale must be"), (dict(scales=torch.ones(4, dtype=torch.float64)), "scale must be"),
    (dict(), "CUDA tensors")])
def test_binding_refuses(changes, message):
    import gemm_kernels as gk

    with pytest.raises(RuntimeError, match=message):
        gk._C.gemm_lora(**{**tensors(), **changes})


def test_binding_refuses_other_shapes_and_types():
    import gemm_kernels as gk

    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        gk._C.gemm_lora(**tensors(dt=torch.float32))
    with pytest.raises(RuntimeError, match="rank must be"):
        gk._C.gemm_lora(**tensors(R=12))
    with pytest.raises(RuntimeError, match="rank must be"):
        gk._C.gemm_lora(**tensors(R=136))
    with pytest.raises(RuntimeError, match="multiple of 8"):
        gk._C.gemm_lora(**tensors(K=124))
    with pytest.raises(ValueError, match="1D"):
        gk.LoraPlan(torch.zeros(3, 3, dtype=torch.int32), 4)
    with pytest.raises(ValueError, match="num_adapters"):
        gk.LoraPlan(torch.zeros(3, dtype=torch.int32), 0)
    with pytest.raises(ValueError, match="CUDA"):
        gk.LoraPlan(torch.zeros(3, dtype=torch.int32), 4)
    with pytest.raises(RuntimeError, match="int32 or int64"):
        gk._C.lora_plan(torch.zeros(3, dtype=torch.int16), 4, torch.zeros(8, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="contiguous"):
        gk._C.lora_plan(torch.zeros(6, dtype=torch.int32)[::2], 4, torch.zeros(8, dtype=torch.uint8))


@pytest.mark.parametrize("changes,want", [(dict(A=None), NULL), (dict(down=None), NULL), (dict(down=0x3008), ALIGN)])
def test_backward_refuses_what_recomputing_needs(lora, changes, want):
    err = I(0)
    assert lora.gemm_sm100_lora_backward(ctypes.byref(good(**changes)), 0x6000, 64, 0x7000, 16, 1, None, 16, None, 128, None, 0xB000,
                                         None, ctypes.byref(err)) == want


@pytest.mark.parametrize("shape,gradient,chosen", [
    # M, N, K, R, adapters of the products, and what carries them out on 148 SMs; every branch of both rules has a line, and each
    # of these shapes is also multiplied on the GPU
    ((5, 4096, 512, 16, 5), False, "few rows: config=13 ctas=64"), ((40, 2048, 1024, 24, 40), False, "few rows: config=14 ctas=32"),
    ((100, 9600, 256, 8, 60), False, "few rows: config=12 ctas=75"), ((128, 1152, 4096, 16, 9), False, "few rows: config=12/4 ctas=36"),
    ((64, 4096, 8448, 16, 3), False, "few rows: config=2/4 ctas=64"), ((9, 136, 8192, 16, 9), False, "few rows: config=12/4 ctas=8"),
    ((256, 9216, 128, 16, 9), False, "less than a wave: config=0 ctas=72"), ((300, 4104, 2000, 24, 30), False, "less than a wave: config=0 ctas=68"),
    ((256, 4480, 8192, 8, 5), False, "less than a wave: config=11 ctas=70"), ((300, 1000, 4096, 24, 30), False, "less than a wave: config=11/2 ctas=64"),
    ((300, 1000, 4096, 24, 30), True, "less than a wave: config=0 ctas=64"), ((250, 264, 8704, 16, 9), True, "less than a wave: config=0 ctas=68"),
    ((300, 4104, 2000, 24, 30), True, "less than a wave: config=0/2 ctas=64"), ((520, 8200, 640, 16, 12), True, "less than a wave: config=2/4 ctas=60"),
    ((256, 8704, 128, 16, 9), False, "planner"), ((2048, 4096, 4096, 32, 8), False, "planner"), ((40, 264, 200, 24, 12), False, "planner"),
    ((256, 9216, 128, 16, 9), True, "planner"),
])
def test_chosen_tiles(shape, gradient, chosen):
    import re

    import gemm_kernels as gk

    rule, words = gk.describe_lora_plan(*shape, gradient=gradient).split(": ", 1)
    cut = re.search(r"cut into (\d+) K ranges", words)
    got = f"{rule}: config={re.search(r'config=([0-9]+)', words)[1]}{'/' + cut[1] if cut else ''} ctas={re.search(r'ctas=([0-9]+)', words)[1]}"
    assert rule == "planner" if chosen == "planner" else got == chosen, got


@pytest.mark.parametrize("shape,gradient", [((0, 64, 64, 8, 1), False), ((8, 0, 64, 8, 1), False), ((8, 64, 60, 8, 1), False),
                                            ((8, 64, 64, 12, 1), False), ((8, 64, 64, 8, 0), False), ((8, 60, 64, 8, 1), True)])
def test_chosen_tiles_refuses(shape, gradient):
    import gemm_kernels as gk

    with pytest.raises(RuntimeError, match="bad shape"):
        gk.describe_lora_plan(*shape, gradient=gradient)


@pytest.mark.parametrize("shape,gradient", [((8192, 64, 1024, 64, 1), False), ((9000, 64, 512, 16, 16), False), ((4096, 64, 8192, 32, 4), False),
                                            ((2048, 1024, 1024, 32, 4), False), ((9000, 1024, 64, 64, 1), True), ((2000, 16384, 256, 16, 16), True),
                                            ((1025, 2048, 512, 16, 4), False)])
def test_many_rows_are_left_to_the_planner(shape, gradient):
    import gemm_kernels as gk

    assert gk.describe_lora_plan(*shape, gradient=gradient).startswith("planner: ")


@pytest.mark.parametrize("shape", [(256, 1536, 8192, 16, 16), (512, 768, 8192, 64, 1), (768, 512, 4096, 32, 4), (600, 504, 4096, 16, 3)])
def test_twelve_narrow_tiles_are_left_to_the_planner(shape):
    import gemm_kernels as gk

    assert gk.describe_lora_plan(*shape).startswith("planner: ")


@pytest.mark.parametrize("shape,gradient,low", [
    # the deep ring where the product behind finds no room beside the short one either
    ((64, 8192, 14336, 64, 16), False, "64 ctas in clusters of 8, deep"), ((1100, 2048, 8192, 64, 1), False, "72 ctas in clusters of 8, deep"),
    ((16, 8192, 8192, 64, 8), False, "32 ctas in clusters of 8, short"), ((700, 1024, 8192, 64, 1), False, "48 ctas in clusters of 8, short"),
    ((512, 4096, 8192, 64, 1), False, "32 ctas in clusters of 8, short"), ((64, 4096, 14336, 64, 32), False, "128 ctas in clusters of 8, short"),
    ((128, 14336, 4096, 16, 64), False, "64 ctas in clusters of 8, short"), ((1100, 8192, 2048, 64, 1), True, "72 ctas in clusters of 8, deep"),
    ((64, 14336, 2048, 64, 16), True, "64 ctas in clusters of 8, short"),
    # (the clusters of a product that is cut along K want more of it), or where few CTAs and the product both have their own SMs
    ((128, 4096, 8192, 64, 8), False, "32 ctas in clusters of 8, deep"), ((128, 8192, 8192, 64, 8), False, "32 ctas in clusters of 8, short"),
    ((66, 27248, 8160, 88, 2), True, "16 ctas in clusters of 8, deep"), ((300, 4096, 8192, 64, 1), False, "24 ctas in clusters of 8, short"),
])
def test_ring_of_the_low_rows(shape, gradient, low):
    import gemm_kernels as gk

    assert gk.describe_lora_plan(*shape, gradient=gradient).endswith(f"; low rows: {low} ring")


@pytest.mark.parametrize("shape,chosen", [
    # tiles of few rows and a long K, by the SMs that the low rows' CTAs (two to an SM) leave
    ((64, 4096, 14336, 64, 32), "config=2 "), ((64, 3584, 14336, 64, 16), "config=2 "), ((64, 3200, 8704, 64, 28), "config=2 "),
    ((16, 3968, 14336, 16, 1), "config=12 "), ((128, 3584, 14336, 16, 8), "config=12 "), ((64, 4096, 14336, 64, 64), "config=12 "),
    ((64, 512, 8704, 64, 28), "config=12 "), ((128, 4224, 28672, 16, 1), "config=2 "),
    ((64, 8448, 17408, 64, 64), "config=2 "),
])
def test_few_rows_beside_the_low_rows(shape, chosen):
    import gemm_kernels as gk

    assert gk.describe_lora_plan(*shape).startswith("few rows: " + chosen)


def test_ring_option():
    import gemm_kernels as gk

    try:
        for value, words in ((1, "deep ring"), (0, "short ring"), (-1, "short ring")):
            gk.set_option("lora_ring", value)
            assert gk.describe_lora_plan(700, 1024, 8192, 64, 1).endswith(words)
        for value in (-2, 2):
            with pytest.raises(RuntimeError, match="unknown option or value"):
                gk.set_option("lora_ring", value)
    finally:
        gk.set_option("lora_ring", -1)


@pytest.mark.parametrize("shape,want", [((1166, 8192, 1704, 24, 9), "less than a wave: config=0 "), ((1792, 1024, 1280, 16, 1), "less than a wave: config=0 "),
                                        ((1045, 344, 1776, 64, 23), "less than a wave: config=0 "), ((1793, 1024, 1024, 16, 1), "planner: "),
                                        ((1100, 14336, 1792, 16, 1), "planner: "), ((1024, 14336, 2304, 16, 1), "less than a wave: config=0 ")])
def test_gradients_of_some_more_rows(shape, want):
    import gemm_kernels as gk

    assert gk.describe_lora_plan(*shape, gradient=True).startswith(want)
