"""Low-rank adapters beside a shared projection, on the GPU, against the definition in 64 bits.

Tolerances, element by element, from the arithmetic the kernels are allowed (u = half a step of the
16-bit type relative to the value, tiny = half its smallest subnormal):
  * a sum of L products accumulated in 32 bits is off by at most  acc(L) = (L + 8) 2^-23  times the sum of
    the products' magnitudes (one addition per product, each off by at most one unit in the last
    place of fp32, which covers truncating adders);
  * low (d_low) is such a sum, rounded once:  d = u |low| + acc(K) sum |A||down| s + tiny;
  * C is a sum of K + R products, rounded once, on low rows that are off by d:
    u |C| + acc(K + R) (sum |A||B| + sum |low||up|) + sum d |up| + tiny;
  * the adapters' gradients are sums over the adapter's rows of products with the rounded rows.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


@pytest.fixture(scope="module")
def gk():
    import gemm_kernels

    return gemm_kernels


def acc(length):
    return (length + 8) * 2.0 ** -23


def make(M, N, K, R, G, dtype, seed, ids):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    t = {"A": normal(M, K, std=1.0), "B": normal(N, K, std=K ** -0.5), "down": normal(G, R, K, std=K ** -0.5),
         "up": normal(G, N, R, std=0.5 * R ** -0.5), "dC": normal(M, N, std=0.5)}
    t["scale"] = 0.5 + 1.5 * torch.rand(G, generator=gen, device="cuda")
    t["ids"] = torch.as_tensor(ids, dtype=torch.int32, device="cuda")
    return t


def id_pattern(kind, M, G, seed):
    gen = torch.Generator().manual_seed(seed + 1000)
    if kind == "one":
        return torch.full((M,), G - 1, dtype=torch.int32)
    if kind == "none":
        return torch.full((M,), -1, dtype=torch.int32)
    if kind == "random":                                   # any order, some rows without, some ids out of range
        ids = torch.randint(-1, G, (M,), generator=gen, dtype=torch.int32)
        ids[torch.rand(M, generator=gen) < 0.03] = G + 5
        ids[torch.rand(M, generator=gen) < 0.03] = -7
        return ids
    if kind == "own":                                      # a row's adapter is its own as long as there are adapters
        return torch.randperm(max(M, G), generator=gen)[:M].to(torch.int32) % G
    assert kind == "runs"                                  # ragged requests one after another
    cuts = sorted(torch.randint(0, M + 1, (6,), generator=gen).tolist())
    ids = torch.empty(M, dtype=torch.int32)
    for i, (a, b) in enumerate(zip([0] + cuts, cuts + [M])):
        ids[a:b] = -1 if i == 3 else int(torch.randint(0, G, (1,), generator=gen))
    return ids


def want(t, low=None):
    """Every result and its bound in 64 bits; `low` replaces the exact rows in the bound of d_up."""
    dtype = t["A"].dtype
    u, tiny = HALF_STEP[dtype], TINY[dtype]
    A, B, dC = t["A"].double(), t["B"].double(), t["dC"].double()
    ids = t["ids"].long()
    M, K = A.shape
    N = B.shape[0]
    G, R = t["down"].shape[:2]
    z = lambda *s: torch.zeros(s, dtype=torch.float64, device="cuda")  # noqa: E731
    res = {"low": z(M, R), "C": A @ B.T, "dA": dC @ B, "d_down": z(G, R, K), "d_up": z(G, N, R)}
    mag = {"low": z(M, R), "C": A.abs() @ B.abs().T, "dA": dC.abs() @ B.abs()}
    d_low, d_mag = z(M, R), z(M, R)
    tol = {"d_down": z(G, R, K) + tiny, "d_up": z(G, N, R) + tiny}
    carried_c, carried_a = z(M, N), z(M, K)
    for g in range(G):
        rows = (ids == g).nonzero().flatten()
        if rows.numel() == 0:
            continue
        down, up, s = t["down"][g].double(), t["up"][g].double(), t["scale"][g].double()
        a, dy = A[rows], dC[rows]
        l, lm = s * a @ down.T, s * a.abs() @ down.abs().T
        dl, dlm = s * dy @ up, s * dy.abs() @ up.abs()
        res["low"][rows], mag["low"][rows] = l, lm
        d_low[rows], d_mag[rows] = dl, dlm
        l_off = u * l.abs() + acc(K) * lm + tiny
        dl_off = u * dl.abs() + acc(N) * dlm + tiny
        res["C"][rows] += l @ up.T
        mag["C"][rows] += l.abs() @ up.abs().T
        carried_c[rows] = l_off @ up.abs().T
        res["dA"][rows] += dl @ down
        mag["dA"][rows] += dl.abs() @ down.abs()
        carried_a[rows] = dl_off @ down.abs()
        n = rows.numel()
        res["d_down"][g] = dl.T @ a
        res["d_up"][g] = dy.T @ l
        tol["d_down"][g] += u * res["d_down"][g].abs() + acc(n) * (dl.abs().T @ a.abs()) + dl_off.T @ a.abs()
        tol["d_up"][g] += u * res["d_up"][g].abs() + acc(n) * (dy.abs().T @ l.abs()) + dy.abs().T @ l_off
    tol["low"] = u * res["low"].abs() + acc(K) * mag["low"] + tiny
    tol["C"] = u * res["C"].abs() + acc(K + R) * mag["C"] + carried_c + tiny
    tol["dA"] = u * res["dA"].abs() + acc(N + R) * mag["dA"] + carried_a + tiny
    # second-order terms (the rounding of a value that is itself off): one part in a hundred covers them
    return res, {k: 1.01 * v for k, v in tol.items()}


def check(name, got, res, tol):
    got = got.double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - res[name]).abs() - tol[name]
    at = int(over.argmax())
    assert float(over.max()) <= 0, (f"{name}: element {at} of {tuple(got.shape)} is {float(got.flatten()[at])}, "
                                    f"should be {float(res[name].flatten()[at])} within {float(tol[name].flatten()[at])}")


def run_all(gk, t):
    plan = gk.LoraPlan(t["ids"], t["down"].shape[0])
    low = torch.full((t["A"].shape[0], t["down"].shape[1]), float("nan"), dtype=t["A"].dtype, device="cuda")
    C = gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low)
    grads = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low)
    gk.device_status()
    return dict(zip(("C", "low", "dA", "d_down", "d_up"), (C, low) + tuple(grads)))


CASES = [
    # M, N, K, R, G, ids
    (1, 64, 64, 8, 1, "one"), (1, 1000, 264, 16, 3, "own"), (2, 8, 8, 8, 2, "own"), (5, 4096, 512, 16, 4, "own"),
    (16, 520, 1032, 24, 16, "own"), (17, 264, 2048, 40, 7, "random"), (64, 1024, 1024, 64, 64, "own"),
    (127, 136, 520, 128, 5, "random"), (128, 512, 256, 16, 128, "own"), (129, 256, 320, 32, 9, "random"),
    (255, 512, 128, 8, 255, "own"), (256, 256, 64, 56, 2, "runs"), (257, 776, 1000, 72, 3, "runs"),
    (300, 1000, 520, 8, 3, "runs"), (513, 264, 72, 16, 300, "random"), (700, 1536, 768, 16, 1, "one"),
    (1025, 512, 1024, 128, 2, "runs"), (1100, 384, 640, 88, 33, "random"), (1500, 256, 256, 32, 600, "own"),
    (2048, 1024, 512, 64, 6, "runs"), (384, 640, 192, 16, 4, "none"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,R,G,kind", CASES)
def test_forward_and_gradients_against_the_definition(gk, M, N, K, R, G, kind, dtype):
    t = make(M, N, K, R, G, dtype, 7 * M + R, id_pattern(kind, M, G, M + N))
    got = run_all(gk, t)
    res, tol = want(t)
    for name, value in got.items():
        check(name, value, res, tol)
