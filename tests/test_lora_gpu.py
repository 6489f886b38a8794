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


@pytest.fixture
def options(gk):
    changed = []

    def set_option(name, value):
        changed.append(name)
        gk.set_option(name, value)

    yield set_option
    defaults = {"tile_config": -1, "split_k": -1, "sk_cluster": -1, "tiles_n": 0, "max_ctas": 0}
    for name in changed:
        gk.set_option(name, defaults[name])


def forward_only(gk, t, **kw):
    plan = gk.LoraPlan(t["ids"], t["down"].shape[0])
    return gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], **kw)


FORCED = [
    # tile configuration, split_k, M, N, K, R, G
    (0, 0, 600, 776, 320, 24, 5), (0, 2, 300, 520, 2048, 16, 9), (0, 4, 300, 520, 4096, 96, 3), (1, 0, 700, 1504, 200, 40, 4),
    (2, 0, 300, 520, 320, 16, 7), (2, 2, 200, 520, 2048, 64, 40), (2, 4, 129, 264, 2112, 128, 6), (9, 0, 16, 1000, 264, 16, 16),
    (10, 0, 64, 520, 328, 72, 30), (11, 0, 300, 648, 640, 8, 12), (11, 2, 257, 264, 2048, 32, 11), (12, 0, 128, 520, 640, 48, 90),
    (12, 4, 100, 392, 4096, 16, 100), (12, 2, 100, 392, 2048, 80, 4), (13, 0, 16, 648, 576, 8, 16), (14, 0, 63, 648, 576, 128, 20), (3, 0, 140, 392, 328, 24, 7),
    (7, 0, 300, 520, 392, 40, 5),
    (14, 0, 64, 200, 256, 16, 64), (15, 0, 9, 776, 640, 104, 4),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("config,split,M,N,K,R,G", FORCED)
def test_every_tile_configuration(gk, options, config, split, M, N, K, R, G, dtype):
    t = make(M, N, K, R, G, dtype, 31 + config, id_pattern("random", M, G, config))
    options("tile_config", config)
    options("split_k", split)
    options("sk_cluster", 1)
    C = forward_only(gk, t)
    gk.device_status()
    res, tol = want(t)
    check("C", C, res, tol)


@pytest.mark.parametrize("config", [0, 1, 2, 3])
@pytest.mark.parametrize("M,N,K,R,G", [(300, 264, 520, 16, 7), (600, 128, 1032, 72, 3), (100, 520, 264, 128, 50)])
def test_every_tile_configuration_of_the_gradient(gk, options, config, M, N, K, R, G):
    t = make(M, N, K, R, G, torch.bfloat16, 57 + config, id_pattern("random", M, G, config))
    options("tile_config", config)
    got = run_all(gk, t)
    gk.device_status()
    res, tol = want(t)
    check("dA", got["dA"], res, tol)


@pytest.mark.parametrize("config,tiles_n,N", [(1, 5, 2240), (0, 5, 1216), (2, 5, 1216)])
def test_balanced_column_tiling(gk, options, config, tiles_n, N):
    t = make(520, N, 256, 24, 4, torch.bfloat16, 71, id_pattern("runs", 520, 4, 3))
    options("tile_config", config)
    options("split_k", 0)
    options("tiles_n", tiles_n)
    C = forward_only(gk, t)
    gk.device_status()
    res, tol = want(t)
    check("C", C, res, tol)


@pytest.mark.parametrize("max_ctas", [2, 6])
def test_many_tiles_per_cta(gk, options, max_ctas):
    t = make(1500, 1544, 192, 40, 5, torch.bfloat16, 73, id_pattern("random", 1500, 5, 4))
    options("max_ctas", max_ctas)
    got = run_all(gk, t)
    gk.device_status()
    res, tol = want(t)
    check("C", got["C"], res, tol)
    check("dA", got["dA"], res, tol)


@pytest.mark.parametrize("M,G,kind", [(96, 40, "own"), (1000, 4, "runs"), (700, 9, "random")])
def test_broken_adapters_and_rows_stay_with_their_own(gk, M, G, kind):
    """Inf and NaN in one adapter's weights and in its rows: every other row, and every other adapter's
    gradient, keeps its bits."""
    N, K, R = 520, 328, 16
    t = make(M, N, K, R, G, torch.bfloat16, 5, id_pattern(kind, M, G, 6))
    clean = run_all(gk, t)
    bad = int(t["ids"][M // 2])
    if not 0 <= bad < G:
        bad = int(t["ids"][(t["ids"] >= 0) & (t["ids"] < G)][0])
    theirs = t["ids"] == bad
    broken = dict(t, A=t["A"].clone(), dC=t["dC"].clone(), down=t["down"].clone(), up=t["up"].clone())
    broken["down"][bad, 3] = float("nan")
    broken["up"][bad, :, 1] = float("inf")
    rows = theirs.nonzero().flatten()
    broken["A"][rows[0]] = float("nan")
    broken["dC"][rows[-1]] = float("inf")
    got = run_all(gk, broken)
    others = torch.arange(G, device="cuda") != bad
    for name in ("C", "low", "dA"):
        assert torch.equal(got[name][~theirs], clean[name][~theirs]), name
    for name in ("d_down", "d_up"):
        assert torch.equal(got[name][others], clean[name][others]), name
    assert not torch.isfinite(got["C"][theirs].float()).all()


def test_rows_without_adapter_equal_the_plain_product(gk):
    t = make(700, 1032, 512, 16, 4, torch.bfloat16, 8, id_pattern("runs", 700, 4, 2))
    C = forward_only(gk, t)
    plain = gk.gemm_tn(t["A"], t["B"])
    none = (t["ids"] < 0) | (t["ids"] >= 4)
    assert bool(none.any()) and torch.equal(C[none], plain[none])
    t["ids"].fill_(-1)
    assert torch.equal(forward_only(gk, t), plain)


def test_strided_operands_and_untouched_neighbours(gk):
    """Row and adapter pitches larger than the rows; nothing outside the outputs is written."""
    M, N, K, R, G = 333, 397, 264, 24, 5
    t = make(M, N + 3, K, R, G, torch.float16, 9, id_pattern("random", M, G, 1))
    wide = {}
    for name, shape in (("A", (M, K)), ("B", (N, K)), ("down", (G, R, K)), ("up", (G, N, R))):
        big = torch.full([s + 8 for s in shape], float("nan"), dtype=torch.float16, device="cuda")
        view = big[tuple(slice(0, s) for s in shape)]
        view.copy_(t[name][tuple(slice(0, s) for s in shape)])
        wide[name] = view
    out = torch.full((M + 2, 416), 7.0, dtype=torch.float16, device="cuda")
    low = torch.full((M + 1, 40), 5.0, dtype=torch.float16, device="cuda")
    plan = gk.LoraPlan(t["ids"].long(), G)
    got = gk.gemm_lora(wide["A"], wide["B"], wide["down"], wide["up"], plan, scale=t["scale"], out=out[:M, :N], low=low[:M, :R])
    assert got.data_ptr() == out.data_ptr()
    t["B"], t["up"], t["dC"] = t["B"][:N], t["up"][:, :N], t["dC"][:, :N]
    res, tol = want(t)
    check("C", got, res, tol)
    check("low", low[:M, :R], res, tol)
    assert bool((out[:, N:] == 7).all()) and bool((out[M:] == 7).all())
    assert bool((low[:, R:] == 5).all()) and bool((low[M:] == 5).all())


def test_same_bits_on_every_call(gk):
    t = make(900, 520, 1024, 32, 6, torch.bfloat16, 10, id_pattern("random", 900, 6, 1))
    first = run_all(gk, t)
    for _ in range(3):
        again = run_all(gk, t)
        for name in first:
            assert torch.equal(first[name], again[name]), name


@pytest.mark.parametrize("needs", [(True, False, False), (False, True, False), (False, False, True), (False, False, False)])
def test_only_the_wanted_gradients(gk, needs):
    t = make(300, 264, 200, 16, 3, torch.bfloat16, 11, id_pattern("runs", 300, 3, 1))
    plan = gk.LoraPlan(t["ids"], 3)
    full = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"])
    some = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], needs=needs)
    for want_it, a, b in zip(needs, full, some):
        assert torch.equal(a, b) if want_it else b is None


def test_number_as_scale_and_kept_low_rows(gk):
    t = make(200, 264, 200, 16, 3, torch.bfloat16, 12, id_pattern("random", 200, 3, 1))
    t["scale"] = torch.full((3,), 0.75, device="cuda")
    plan = gk.LoraPlan(t["ids"], 3)
    low = torch.empty(200, 16, dtype=torch.bfloat16, device="cuda")
    a = gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=0.75, low=low)
    assert torch.equal(a, forward_only(gk, t))
    kept = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=0.75, low=low)
    again = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=0.75)
    for x, y in zip(kept, again):
        assert torch.equal(x, y)


def test_empty_batch(gk):
    t = make(0, 264, 200, 16, 3, torch.bfloat16, 13, torch.empty(0))
    got = run_all(gk, t)
    assert got["C"].shape == (0, 264) and got["dA"].shape == (0, 200)
    assert bool((got["d_down"] == 0).all()) and bool((got["d_up"] == 0).all())


def test_captured_step_follows_the_plan(gk):
    """Forward and backward captured with the plan's update; replays with other ids and inputs give what the
    eager calls give, also with two captured graphs that run side by side."""
    M, N, K, R, G = 500, 520, 512, 16, 6
    batches = [make(M, N, K, R, G, torch.bfloat16, 20 + i, id_pattern(kind, M, G, i))
               for i, kind in enumerate(("runs", "random", "own"))]
    eager = [run_all(gk, t) for t in batches]
    graphs = []
    for _ in range(2):
        s = {k: v.clone() for k, v in batches[0].items()}
        plan = gk.LoraPlan(s["ids"], G)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.update(s["ids"])
            low = torch.empty(M, R, dtype=torch.bfloat16, device="cuda")
            C = gk.gemm_lora(s["A"], s["B"], s["down"], s["up"], plan, scale=s["scale"], low=low)
            grads = gk.gemm_lora_backward(s["dC"], s["A"], s["B"], s["down"], s["up"], plan, scale=s["scale"])
        graphs.append((s, graph, dict(zip(("C", "low", "dA", "d_down", "d_up"), (C, low) + grads))))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for first, second in ((0, 1), (1, 2), (2, 0)):
        torch.cuda.synchronize()
        for (s, _, _), i in zip(graphs, (first, second)):
            for k, v in batches[i].items():
                s[k].copy_(v)
        torch.cuda.synchronize()
        for (_, graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, out), i in zip(graphs, (first, second)):
            for name, value in out.items():
                assert torch.equal(value, eager[i][name]), (name, i)
    gk.device_status()


def test_two_streams_at_once(gk):
    t = [make(400, 776, 1024, 32, 5, torch.bfloat16, 30 + i, id_pattern("random", 400, 5, i)) for i in range(2)]
    alone = [run_all(gk, x) for x in t]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for _ in range(5):
        for s, x in zip(streams, t):
            with torch.cuda.stream(s):
                results.append(run_all(gk, x))
    torch.cuda.synchronize()
    for i, got in enumerate(results):
        for name in got:
            assert torch.equal(got[name], alone[i % 2][name]), name


def test_a_plan_outlives_its_last_reference(gk):
    """A plan made on one stream and used on another may be dropped while the kernels that read it are queued."""
    t = make(300, 520, 1024, 16, 4, torch.bfloat16, 40, id_pattern("random", 300, 4, 1))
    alone = forward_only(gk, t)
    side = torch.cuda.Stream()
    plan = gk.LoraPlan(t["ids"], 4)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-4
        got = gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"])
    size = plan.buffer.numel()
    del plan
    torch.full((size,), 255, dtype=torch.uint8, device="cuda")     # would take the freed block
    torch.cuda.synchronize()
    assert torch.equal(got, alone)


def test_gradients_against_differences(gk):
    """Central differences of the plain 64-bit forward pass along random directions."""
    M, N, K, R, G = 40, 64, 48, 8, 3
    t = make(M, N, K, R, G, torch.float16, 50, id_pattern("random", M, G, 2))
    got = run_all(gk, t)
    ids, valid = t["ids"].long(), (t["ids"] >= 0) & (t["ids"] < G)
    x = {k: t[k].double() for k in ("A", "B", "down", "up", "dC", "scale")}

    def loss(A, down, up):
        total = (A @ x["B"].T * x["dC"]).sum()
        for m in valid.nonzero().flatten().tolist():
            g = int(ids[m])
            total = total + (x["scale"][g] * (up[g] @ (down[g] @ A[m])) * x["dC"][m]).sum()
        return total

    gen = torch.Generator(device="cuda").manual_seed(3)
    for i, name in enumerate(("A", "down", "up")):
        direction = torch.randn(x[name].shape, generator=gen, device="cuda", dtype=torch.float64)
        args = [x["A"], x["down"], x["up"]]
        step = 1e-3
        up_args, down_args = list(args), list(args)
        up_args[i], down_args[i] = args[i] + step * direction, args[i] - step * direction
        slope = float((loss(*up_args) - loss(*down_args)) / (2 * step))
        grad = got["dA" if name == "A" else "d_" + name].double()
        # the loss is linear in each argument, so the difference is exact but for 64-bit rounding; each
        # element of the gradient carries its own tolerance
        _, tol = want(t)
        bound = float((tol["dA" if name == "A" else "d_" + name] * direction.abs()).sum()) + 1e-6
        assert abs(float((grad * direction).sum()) - slope) <= bound


@pytest.mark.parametrize("M,G,kind", [(1, 1, "one"), (255, 30, "random"), (256, 256, "own"), (700, 9, "random"), (1000, 4096, "own"),
                                      (513, 5, "none")])
@pytest.mark.parametrize("wide", [False, True])
def test_plan_contents(gk, M, G, kind, wide):
    """The slot lists, row masks and per-adapter row lists against a plain construction."""
    ids = id_pattern(kind, M, G, M)
    if wide:
        ids = ids.long()
        ids[ids < 0] = 2 ** 40 + 1                          # no adapter, although its low 32 bits are 1
    plan = gk.LoraPlan(ids.cuda(), G)
    words = plan.buffer.view(torch.int32).cpu().tolist()
    up64 = lambda n: (n + 63) // 64 * 64  # noqa: E731
    tiles = -(-M // 256)
    at = up64(tiles)
    adapters, masks = at, at + tiles * 256
    row_slot = masks + tiles * 256 * 8
    order = row_slot + up64(M)
    offsets = order + up64(M)
    clean = [i if 0 <= i < G else -1 for i in ids.tolist()]
    for t in range(tiles):
        rows = clean[t * 256:(t + 1) * 256]
        slots = list(dict.fromkeys(i for i in rows if i >= 0))
        assert words[t] == len(slots)
        assert words[adapters + t * 256:adapters + t * 256 + len(slots)] == slots
        for j, g in enumerate(slots):
            mask = sum(1 << r for r, i in enumerate(rows) if i == g)
            got = words[masks + (t * 256 + j) * 8:masks + (t * 256 + j) * 8 + 8]
            assert sum((w & 0xffffffff) << (32 * k) for k, w in enumerate(got)) == mask
        assert words[row_slot + t * 256:row_slot + t * 256 + len(rows)] == [slots.index(i) if i >= 0 else -1 for i in rows]
    want_order = [m for g in sorted(set(clean) - {-1}) for m in range(M) if clean[m] == g]
    assert words[order:order + len(want_order)] == want_order
    counts = [0] * G
    for i in clean:
        if i >= 0:
            counts[i] += 1
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    assert words[offsets:offsets + G + 1] == starts


@pytest.mark.parametrize("N", [1, 3, 9, 63])
def test_columns_that_fill_no_piece(gk, N):
    """A handful of columns inside a wider buffer: the columns behind them keep what they held."""
    M, K, R, G = 70, 72, 8, 3
    t = make(M, 64, K, R, G, torch.bfloat16, 60 + N, id_pattern("random", M, G, 5))
    t["B"], t["up"], t["dC"] = t["B"][:N], t["up"][:, :N].contiguous(), t["dC"][:, :N]
    out = torch.full((M, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    forward_only(gk, t, out=out[:, :N])
    res, tol = want(t)
    check("C", out[:, :N], res, tol)
    assert bool((out[:, N:] == 3).all())


def test_first_use_inside_a_capture():
    """In a fresh process: init(), then a plan, a forward and a backward pass captured as the first calls of all."""
    import os
    import subprocess
    import sys

    code = """
import sys; sys.path[:0] = [{repo!r}, {pkg!r}]
import torch, gemm_kernels as gk
gk.init()
dt, M, N, K, R, G = torch.bfloat16, 200, 264, 320, 24, 5
r = lambda *s: torch.randn(*s, device="cuda").to(dt)
A, B, down, up, dC = r(M, K), r(N, K), r(G, R, K), r(G, N, R), r(M, N)
ids = torch.arange(M, device="cuda", dtype=torch.int32) % G
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    plan = gk.LoraPlan(ids, G)
    C = gk.gemm_lora(A, B, down, up, plan)
    grads = gk.gemm_lora_backward(dC, A, B, down, up, plan)
graph.replay()
torch.cuda.synchronize()
plan2 = gk.LoraPlan(ids, G)
assert torch.equal(C, gk.gemm_lora(A, B, down, up, plan2))
for x, y in zip(grads, gk.gemm_lora_backward(dC, A, B, down, up, plan2)):
    assert torch.equal(x, y)
gk.device_status()
print("captured")
"""
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = subprocess.run([sys.executable, "-c", code.format(repo=repo, pkg=os.path.join(repo, "cute-examples_b200"))],
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_one_step_after_another(gk):
    """A run as a training loop makes it: plan refilled, forward, backward, the adapters updated in place, twice, next
    to plain products of the library; against the same loop in 64 bits within the first step's tolerances."""
    M, N, K, R, G = 512, 264, 328, 16, 3
    t = make(M, N, K, R, G, torch.bfloat16, 80, id_pattern("runs", M, G, 3))
    plan = gk.LoraPlan(t["ids"], G)
    for step in range(2):
        t["ids"] = id_pattern("runs", M, G, 10 + step).cuda()
        plan.update(t["ids"])
        low = torch.empty(M, R, dtype=torch.bfloat16, device="cuda")
        plain = gk.gemm_tn(t["A"], t["B"])
        C = gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low)
        after = gk.gemm_tn(t["A"], t["B"])
        dA, d_down, d_up = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low)
        assert torch.equal(plain, after)
        res, tol = want(t)
        for name, value in (("C", C), ("low", low), ("dA", dA), ("d_down", d_down), ("d_up", d_up)):
            check(name, value, res, tol)
        t["down"] -= 0.01 * d_down
        t["up"] -= 0.01 * d_up
    gk.device_status()


def test_long_rows_and_far_adapters(gk):
    """Offsets that pass 32 bits: adapters whose weights lie more than 4 GiB apart."""
    N, K, R, G, M = 64, 64, 8, 3, 5
    gap = (2 ** 31 + 2 ** 20) // 2                         # elements between adapters: the third starts behind 4 GiB
    big = torch.empty(2 * gap + N * K, dtype=torch.bfloat16, device="cuda")
    t = make(M, N, K, R, G, torch.bfloat16, 90, torch.tensor([2, 0, 1, 2, -1]))
    down = big.as_strided((G, R, K), (gap, K, 1))
    down.copy_(t["down"])
    plan = gk.LoraPlan(t["ids"], G)
    C = gk.gemm_lora(t["A"], t["B"], down, t["up"], plan, scale=t["scale"])
    res, tol = want(t)
    check("C", C, res, tol)
    up = big.as_strided((G, N, R), (gap, R, 1))
    up.copy_(t["up"])
    C = gk.gemm_lora(t["A"], t["B"], t["down"], up, plan, scale=t["scale"])
    check("C", C, res, tol)
    grads = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], up, plan, scale=t["scale"])
    for name, value in zip(("dA", "d_down", "d_up"), grads):
        check(name, value, res, tol)


@pytest.mark.parametrize("M,N,K,R,G", [(5, 4096, 512, 16, 5), (40, 2048, 1024, 24, 40), (100, 9600, 256, 8, 60), (128, 1152, 4096, 16, 9),
                                       (64, 4096, 8448, 64, 20), (64, 4096, 8448, 16, 3), (33, 8448, 17408, 8, 2),
                                       (40, 264, 2048, 24, 12), (3, 8, 1024, 8, 3), (9, 136, 8192, 16, 9)])
def test_few_rows_under_the_own_plan(gk, M, N, K, R, G):
    """A case for each branch of the tile choice for few rows."""
    t = make(M, N, K, R, G, torch.bfloat16, 100 + M, id_pattern("random", M, G, 8))
    C = forward_only(gk, t)
    gk.device_status()
    res, tol = want(t)
    check("C", C, res, tol)


@pytest.mark.parametrize("M,N,K,R,G", [(256, 8704, 128, 16, 9), (256, 4480, 8192, 8, 5), (300, 1000, 4096, 24, 30), (600, 504, 4096, 16, 3),
                                       (250, 264, 8704, 16, 9), (500, 520, 4096, 8, 40), (300, 4104, 2000, 24, 30),
                                       (520, 8200, 640, 16, 12)])
def test_less_than_a_wave_under_the_own_plan(gk, M, N, K, R, G):
    """A case for each branch of the tile choice for outputs of less than a wave: four of the forward product, four of dA."""
    t = make(M, N, K, R, G, torch.bfloat16, 140 + M, id_pattern("random", M, G, 8))
    C = forward_only(gk, t)
    res, tol = want(t)
    check("C", C, res, tol)
    plan = gk.LoraPlan(t["ids"], G)
    grads = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"])
    for name, value in zip(("dA", "d_down", "d_up"), grads):
        check(name, value, res, tol)
    gk.device_status()


def test_plan_refilled_before_every_call(gk):
    """A plan that changes in place just before the product reads it: a stale copy of the old plan, in some SM's cache,
    would give wrong rows or leave the kernel's warps at odds about the number of adapters."""
    M, N, K, R, G = 40, 8192, 256, 16, 40
    t = make(M, N, K, R, G, torch.bfloat16, 120, id_pattern("own", M, G, 1))
    patterns = [id_pattern("own", M, G, 1).cuda(), id_pattern("one", M, G, 1).cuda(), id_pattern("random", M, 5, 2).cuda(),
                id_pattern("none", M, G, 1).cuda(), id_pattern("random", M, G, 3).cuda()]
    wanted = []
    for ids in patterns:
        t["ids"] = ids
        wanted.append(forward_only(gk, t))
    res, tol = want(t)
    check("C", wanted[-1], res, tol)
    plan = gk.LoraPlan(patterns[0], G)
    outs = [torch.empty(M, N, dtype=torch.bfloat16, device="cuda") for _ in range(8)]
    for step in range(0, 400, 8):
        for i in range(8):
            plan.update(patterns[(step + 3 * i) % 5])
            gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], out=outs[i])
        for i in range(8):
            assert torch.equal(outs[i], wanted[(step + 3 * i) % 5]), (step, i)
    gk.device_status()


@pytest.mark.parametrize("M,N,K,R", [(5, 4096, 512, 16), (7, 20320, 320, 24), (3, 1024, 64, 8), (100, 512, 64, 16), (300, 776, 64, 24)])
def test_short_main_loops_many_times(gk, M, N, K, R):
    """A main loop of one or two ring stages: the plan's entries are needed almost at once.  Fresh plans and inputs
    every time, as the first pass over a new batch has them."""
    G = 9
    for seed in range(40):
        t = make(M, N, K, R, G, torch.bfloat16, 200 + seed, id_pattern("random", M, G, seed))
        torch.empty(1 << 26, dtype=torch.uint8, device="cuda").fill_(seed)      # other data in the caches
        C = forward_only(gk, t)
        res, tol = want(t)
        check("C", C, res, tol)
    gk.device_status()


@pytest.mark.parametrize("M,N,K,R,G,kind", [(70001, 64, 64, 8, 300, "random"), (3, 150000, 64, 16, 3, "own"), (130, 72, 40000, 24, 4, "runs")])
def test_one_long_extent(gk, M, N, K, R, G, kind):
    t = make(M, N, K, R, G, torch.bfloat16, 300, id_pattern(kind, M, G, 9))
    got = run_all(gk, t)
    gk.device_status()
    res, tol = want(t)
    for name, value in got.items():
        check(name, value, res, tol)


def test_threads_that_call_at_once(gk):
    """Four host threads on streams of their own, each with its plans and sizes."""
    import threading

    cases = [make(100 + 60 * i, 264 + 8 * i, 320, 16, 3 + i, torch.bfloat16, 400 + i, id_pattern("random", 100 + 60 * i, 3 + i, i))
             for i in range(4)]
    alone = [run_all(gk, t) for t in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = run_all(gk, cases[i])
                torch.cuda.current_stream().synchronize()
                wrong.extend((i, name) for name in got if not torch.equal(got[name], alone[i][name]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong
    gk.device_status()


def backward_variants(gk, t):
    """The gradients for every way of calling the backward pass: `low` kept or computed again, any of them unwanted."""
    plan = gk.LoraPlan(t["ids"], t["down"].shape[0])
    low = torch.empty(t["A"].shape[0], t["down"].shape[1], dtype=t["A"].dtype, device="cuda")
    gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low)
    for kept in (None, low):
        for bits in range(1, 8):
            needs = tuple(bool(bits >> i & 1) for i in range(3))
            yield needs, gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=kept, needs=needs)


@pytest.mark.parametrize("M,N,K,R,G,kind", [(200, 64, 1024, 16, 3, "runs"), (300, 1024, 128, 16, 3, "runs"), (2500, 1024, 1024, 16, 4, "runs"),
                                            (130, 72, 40000, 24, 4, "runs"), (8192, 512, 1024, 16, 2, "runs"), (700, 264, 1024, 16, 60, "random"),
                                            (3000, 4096, 256, 40, 3, "runs"), (1100, 8, 712, 128, 30, "random")])
def test_kept_and_recomputed_low_rows_give_the_same_bits(gk, M, N, K, R, G, kind):
    """Extents where a launch that low and d_low share has to cut one of them less, or more, than a launch of its own would."""
    t = make(M, N, K, R, G, torch.bfloat16, 500 + M, id_pattern(kind, M, G, 3))
    first = None
    for needs, grads in backward_variants(gk, t):
        first = first or list(grads)
        for i, (wanted, value) in enumerate(zip(needs, grads)):
            if wanted and first[i] is None:
                first[i] = value
            assert torch.equal(value, first[i]) if wanted else value is None, (needs, i)
    res, tol = want(t)
    for name, value in zip(("dA", "d_down", "d_up"), first):
        check(name, value, res, tol)
    gk.device_status()


@pytest.mark.parametrize("M,N,K,R,G,kind", [(1024, 12000, 1032, 64, 1, "one"), (1024, 1032, 12000, 48, 1, "one"), (900, 13000, 264, 128, 3, "runs")])
def test_unwanted_gradients_leave_the_bits_of_the_others(gk, M, N, K, R, G, kind):
    """Extents where one adapter gradient alone has fewer column tiles than the device holds CTAs, and both have more."""
    t = make(M, N, K, R, G, torch.float16, 600 + K, id_pattern(kind, M, G, 3))
    first = None
    for needs, grads in backward_variants(gk, t):
        first = first or list(grads)
        for i, (wanted, value) in enumerate(zip(needs, grads)):
            if wanted and first[i] is None:
                first[i] = value
            assert torch.equal(value, first[i]) if wanted else value is None, (needs, i)
    res, tol = want(t)
    for name, value in zip(("dA", "d_down", "d_up"), first):
        check(name, value, res, tol)
    gk.device_status()


@pytest.mark.parametrize("N", [1, 9, 397])
@pytest.mark.parametrize("M", [1, 2, 70])
@pytest.mark.parametrize("form", ["none", "pitched", "dense"])
def test_columns_that_are_no_multiple_of_8(gk, M, N, form):
    K, R, G = 72, 8, 3
    t = make(M, 400, K, R, G, torch.bfloat16, 700 + N, id_pattern("own", M, G, 5))
    t["B"], t["up"], t["dC"] = t["B"][:N], t["up"][:, :N].contiguous(), t["dC"][:, :N]
    wide = torch.full((M + 1, 416), 3.0, dtype=torch.bfloat16, device="cuda")
    line = torch.full((M * N + 64,), 3.0, dtype=torch.bfloat16, device="cuda")
    out = {"none": None, "pitched": wide[:M, :N], "dense": line[:M * N].view(M, N)}[form]
    if form == "dense" and M > 1:
        with pytest.raises(RuntimeError, match="16-byte aligned"):
            forward_only(gk, t, out=out)
        return
    got = forward_only(gk, t, out=out)
    assert got.shape == (M, N) and got.stride(1) == 1
    assert out is None or got.data_ptr() == out.data_ptr()
    res, tol = want(t)
    check("C", got, res, tol)
    assert bool((wide[:, N:] == 3).all()) and bool((wide[M:] == 3).all()) and bool((line[M * N:] == 3).all())
    again = forward_only(gk, t)
    assert torch.equal(got, again)


def test_widest_output_of_less_than_a_wave(gk):
    """36 pair tiles in one tile row, the fewest that such an output of at most 256 rows keeps whole."""
    t = make(256, 9216, 128, 16, 9, torch.bfloat16, 800, id_pattern("random", 256, 9, 8))
    assert gk.describe_lora_plan(256, 9216, 128, 16, 9).startswith("less than a wave: config=0 ")
    got = run_all(gk, t)
    res, tol = want(t)
    for name, value in got.items():
        check(name, value, res, tol)
    gk.device_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K,R,G,kind,deep", [(16, 8192, 4096, 64, 16, "own", "forward"), (1100, 4096, 2048, 64, 1, "one", "backward"),
                                                 (500, 8192, 2048, 40, 2, "runs", "both in one launch")])
def test_low_rows_through_the_deep_ring(gk, M, N, K, R, G, kind, deep, dtype):
    """The low rows of a forward pass, of a backward pass that kept them, and both kinds in one launch (64 CTAs)."""
    t = make(M, N, K, R, G, dtype, 900 + M, id_pattern(kind, M, G, 3))
    if deep in ("forward", "backward"):
        assert gk.describe_lora_plan(M, N, K, R, G, gradient=deep == "backward").endswith("deep ring")
    res, tol = want(t)
    for name, value in run_all(gk, t).items():
        check(name, value, res, tol)
    plan = gk.LoraPlan(t["ids"], G)
    grads = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"])
    for name, value in zip(("dA", "d_down", "d_up"), grads):
        check(name, value, res, tol)
    gk.device_status()


@pytest.mark.parametrize("M,K,R,G,kind", [(1, 64, 8, 3, "own"), (77, 1032, 24, 5, "random"), (300, 520, 128, 9, "runs"), (2500, 1024, 16, 4, "runs"),
                                          (900, 264, 40, 60, "random"), (64, 14336, 64, 32, "own")])
def test_low_rows_as_a_call_of_their_own(gk, M, K, R, G, kind):
    """gemm_sm100_lora_low without B and up: the rows that a forward pass leaves, bit for bit, also with a pitch."""
    import ctypes

    from conftest import load_capi
    from test_lora_host import LoraArgs

    t = make(M, 72, K, R, G, torch.bfloat16, 1000 + M, id_pattern(kind, M, G, 3))
    plan = gk.LoraPlan(t["ids"], G)
    low = torch.empty(M, R, dtype=torch.bfloat16, device="cuda")
    gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low)
    wide = torch.full((M + 1, R + 16), 3.0, dtype=torch.bfloat16, device="cuda")
    args = LoraArgs(M=M, N=72, K=K, R=R, adapters=G, dtype=0, A=t["A"].data_ptr(), B=None, down=t["down"].data_ptr(), up=None, lda=K, ldb=0,
                    ld_down=K, stride_down=R * K, ld_up=0, stride_up=0, scales=t["scale"].data_ptr(), scale=1.0, plan=plan.buffer.data_ptr())
    err = ctypes.c_int(0)
    call = load_capi().gemm_sm100_lora_low
    call.argtypes = [ctypes.POINTER(LoraArgs), ctypes.c_void_p, ctypes.c_long, ctypes.c_void_p, ctypes.POINTER(ctypes.c_int)]
    assert call(ctypes.byref(args), wide.data_ptr(), R + 16, torch.cuda.current_stream().cuda_stream, ctypes.byref(err)) == 0
    gk.device_status()
    assert torch.equal(wide[:M, :R], low) and bool((wide[:, R:] == 3).all()) and bool((wide[M:] == 3).all())
    res, tol = want(t)
    check("low", low, res, tol)


def test_threads_that_share_a_stream(gk):
    """Four host threads on one stream: any kernel of another thread may stand in front of a product that starts before its
    predecessor has finished.  Plans are refilled in between, and plain products run among them."""
    import threading

    shared = torch.cuda.Stream()
    cases = [[make(90 + 150 * i, 264 + 520 * i, 328 + 64 * i, 16, 3 + i, torch.bfloat16, 1100 + 2 * i + j,
                   id_pattern("random", 90 + 150 * i, 3 + i, j)) for j in range(2)] for i in range(4)]
    alone = [[run_all(gk, t) for t in pair] for pair in cases]
    plain = [[gk.gemm_tn(t["A"], t["B"]) for t in pair] for pair in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(shared):
            plan = gk.LoraPlan(cases[i][0]["ids"], 3 + i)
            for step in range(40):
                j = step % 2
                t = cases[i][j]
                plan.update(t["ids"])
                low = torch.empty(t["A"].shape[0], 16, dtype=torch.bfloat16, device="cuda")
                C = gk.gemm_lora(t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low)
                other = gk.gemm_tn(t["A"], t["B"])
                grads = gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"], low=low if step % 3 else None)
                got = dict(zip(("C", "low", "dA", "d_down", "d_up"), (C, low) + grads))
                same = [torch.equal(v, alone[i][j][name]) for name, v in got.items()] + [torch.equal(other, plain[i][j])]
                if not all(same):
                    wrong.append((i, step, same))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not wrong, wrong[:3]
    gk.device_status()


@pytest.mark.parametrize("M,N,K,R,G,kind", [(1, 64, 64, 8, 1, "one"), (130, 72, 4000, 24, 4, "runs"), (64, 1024, 1024, 64, 64, "own"),
                                            (700, 264, 1024, 16, 60, "random"), (2500, 1024, 1024, 16, 4, "runs"), (300, 200, 264, 128, 9, "random")])
def test_either_ring_gives_the_same_bits(gk, M, N, K, R, G, kind):
    t = make(M, N, K, R, G, torch.bfloat16, 1200 + M, id_pattern(kind, M, G, 3))
    plan = gk.LoraPlan(t["ids"], G)
    got = []
    try:
        for ring in (0, 1):
            gk.set_option("lora_ring", ring)
            got.append(list(run_all(gk, t).values()) +
                       list(gk.gemm_lora_backward(t["dC"], t["A"], t["B"], t["down"], t["up"], plan, scale=t["scale"])))
    finally:
        gk.set_option("lora_ring", -1)
    for a, b in zip(*got):
        assert torch.equal(a, b)
    gk.device_status()
