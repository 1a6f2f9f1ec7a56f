"""Low-rank adapters beside a shared projection and their gradients, against the definition in 64 bits.

Tolerances are bounds, element by element (u = 2^-24, bf16 half step 2^-8): sums of K exact products are off by at most
2 (K + 1) u sum |a b|; the inner product is rounded to bf16 once for bf16 results, and kept to 24 bits (3 u, with its three
summands) for FP32 results; bf16 results are rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -24, 2.0 ** -8
NAN = float("nan")


def make(T, N, D, R, n, order="sorted", nk=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn(T, D, generator=g).bfloat16()
    W = (torch.randn(N, D, generator=g) / D ** 0.5).bfloat16()
    A = (torch.randn(n, R, D, generator=g) / D ** 0.5).bfloat16()
    B = (torch.randn(n, R, N, generator=g) / R ** 0.5).bfloat16()
    s = torch.rand(n, generator=g) + 0.5
    if order == "none":
        ids = torch.full((T,), -1)
    else:
        ids = torch.randint(-1, n, (T,), generator=g)
        if order == "sorted":
            ids = ids.sort()[0]
        elif order == "one":
            ids = torch.full((T,), n - 1)
    if not nk:
        W = W.t().contiguous()
    return X.cuda(), W.cuda(), A.cuda(), B.cuda(), ids.int().cuda(), s.cuda()


def select(p, ids, s, n):
    """[T, n, R] -> the row's own, scaled, zero elsewhere, as [T, n * R]"""
    mine = ids[:, None] == torch.arange(n, device=ids.device)
    return torch.where(mine[..., None], p * s.view(1, n, 1), torch.zeros((), dtype=p.dtype, device=p.device)).flatten(1)


def exact(X, W, A, B, ids, s, nk, f32):
    x, w, a, b = X.double(), (W.t() if nk else W).double(), A.double(), B.double()
    n, R, D = a.shape
    v = select((x @ a.flatten(0, 1).T).view(-1, n, R), ids, s.double(), n)
    va = select((x.abs() @ a.abs().flatten(0, 1).T).view(-1, n, R), ids, s.double().abs(), n)
    bf = b.flatten(0, 1)
    y = x @ w + v @ bf
    ev = (2 * (D + 1) + 2) * U * va + (3 * U if f32 else HALF) * (v.abs() + (2 * D + 4) * U * va)
    tol = 2 * (D + 1 + 4 * R) * U * (x.abs() @ w.abs() + va @ bf.abs()) + ev @ bf.abs() + (U if f32 else HALF) * y.abs()
    return y, 1.02 * tol + 1e-30


def exact_grad(X, dY, A, B, ids, s, f32):
    x, dy, a, b = X.double(), dY.double(), A.double(), B.double()
    n, R, D = a.shape
    N, T = b.shape[2], x.shape[0]
    res = []
    for p, q, m, K in ((dy, x, b, N), (x, dy, a, D)):
        u = select((p @ m.flatten(0, 1).T).view(-1, n, R), ids, s.double(), n)
        ua = select((p.abs() @ m.abs().flatten(0, 1).T).view(-1, n, R), ids, s.double().abs(), n)
        eu = (2 * (K + 1) + 2) * U * ua + (3 * U if f32 else HALF) * (u.abs() + (2 * K + 4) * U * ua)
        g = (u.T @ q).view(n, R, -1)
        tol = (eu.T @ q.abs()).view(n, R, -1) + 2 * (3 * T + 1) * U * (ua.T @ q.abs()).view(n, R, -1) + (U if f32 else HALF) * g.abs()
        res.append((g, 1.02 * tol + 1e-30))
    return res


def within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() / tol).max():.3g} x its bound"


def check(ops, X, W, A, B, ids, s, nk, f32):
    dt = torch.float32 if f32 else torch.bfloat16
    y = ops.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=nk, out_dtype=dt)
    ops.check_status()
    within(y, *exact(X, W, A, B, ids, s, nk, f32), "Y")
    return y


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("nk", [True, False])
@pytest.mark.parametrize("T,N,D,R,n,order", [
    (1, 8, 8, 1, 1, "one"), (1, 512, 264, 16, 4, "one"), (2, 200, 64, 8, 3, "mixed"), (17, 264, 136, 17, 5, "mixed"), (64, 256, 512, 16, 64, "mixed"),
    (65, 1032, 200, 33, 70, "mixed"), (128, 128, 128, 64, 128, "mixed"), (129, 520, 256, 100, 9, "sorted"), (257, 264, 72, 128, 300, "mixed"),
    (300, 512, 256, 16, 40, "none"), (511, 128, 264, 20, 60, "mixed"), (512, 128, 264, 20, 60, "mixed"), (600, 64, 8192, 16, 30, "mixed"),
    (700, 136, 1032, 128, 40, "mixed"), (600, 72, 4104, 50, 30, "sorted"), (32, 264, 4096, 16, 20, "mixed"), (33, 520, 72, 8, 33, "mixed"), (1030, 264, 520, 48, 7, "sorted"), (1100, 128, 1000, 16, 50, "mixed"), (1500, 776, 320, 32, 3, "one"),
])
def test_projection_with_adapters(ops, T, N, D, R, n, order, nk, f32):
    check(ops, *make(T, N, D, R, n, order, nk, seed=T + R), nk, f32)


@pytest.mark.parametrize("f32", [False, True])
def test_split_over_k_shares_the_adapters_out(ops, f32):
    # few tiles and a long K: the K ranges take the adapters in turn
    check(ops, *make(50, 512, 8192, 16, 64, "mixed"), True, f32)
    check(ops, *make(200, 256, 16384, 64, 5, "sorted"), True, f32)


def test_long_k_takes_the_run_time_schedule(ops):
    check(ops, *make(2600, 2304, 6144, 16, 6, "sorted"), True, False)


def test_equals_the_plain_projection_where_no_row_has_an_adapter(ops):
    X, W, A, B, ids, s = make(300, 512, 256, 16, 4, "none")
    assert torch.equal(ops.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=True), ops.gemm_bf16(X, W, b_is_nk=True))
    # and such rows are the plain ones next to rows with adapters, in every tile
    X, W, A, B, ids, s = make(300, 512, 256, 16, 4, "mixed")
    y, p = ops.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=True), ops.gemm_bf16(X, W, b_is_nk=True)
    assert torch.equal(y[ids < 0], p[ids < 0])


def test_scales_default_to_one(ops):
    X, W, A, B, ids, s = make(100, 256, 128, 16, 4, "mixed")
    a = ops.gemm_bf16_lora(X, W, A, B, ids, b_is_nk=True)
    b = ops.gemm_bf16_lora(X, W, A, B, ids, torch.ones_like(s), b_is_nk=True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("T", [60, 300, 1300])
@pytest.mark.parametrize("f32", [False, True])
def test_requests_do_not_reach_each_other(ops, T, f32):
    """NaN and infinities in one adapter, in one token, or an id without an adapter stay in the rows concerned."""
    X, W, A, B, ids, s = make(T, 264, 256, 24, 8, "mixed")
    dt = torch.float32 if f32 else torch.bfloat16
    clean = ops.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=True, out_dtype=dt)
    A2, B2, X2, i2 = A.clone(), B.clone(), X.clone(), ids.clone()
    B2[3, 2] = float("inf")
    B2[4] = NAN
    A2[5, 1, 7] = NAN
    X2[11] = NAN
    i2[13], i2[14] = 8, 2 ** 31 - 1
    y = ops.gemm_bf16_lora(X2, W, A2, B2, i2, s, b_is_nk=True, out_dtype=dt)
    ops.check_status()
    touched = (i2 == 3) | (i2 == 4) | (i2 == 5) | (i2 >= 8)
    touched[11] = True
    assert torch.equal(y[~touched], clean[~touched])
    assert not y[touched].isfinite().any()


def test_strided_operands_and_output(ops):
    T, N, D, R, n = 150, 264, 136, 12, 5
    X, W, A, B, ids, s = make(T, N, D, R, n, "mixed")
    want = ops.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=True)
    Xp, Wp = torch.full((T, D + 8), NAN, device="cuda").bfloat16(), torch.full((N, D + 16), NAN, device="cuda").bfloat16()
    Xp[:, :D], Wp[:, :D] = X, W
    # adapters as slices of stacks of a larger rank (the ranks above are not read)
    Ap, Bp = torch.full((n, R + 4, D + 8), NAN, device="cuda").bfloat16(), torch.full((n, R + 6, N + 8), NAN, device="cuda").bfloat16()
    Ap[:, :R, :D], Bp[:, :R, :N] = A, B
    o = torch.full((T + 5, N + 8), 5.0, device="cuda").bfloat16()
    got = ops.gemm_bf16_lora(Xp[:, :D], Wp[:, :D], Ap[:, :R, :D], Bp[:, :R, :N], ids, s, out=o[:T, :N], b_is_nk=True)
    assert torch.equal(got, want)
    assert (o[T:] == 5).all() and (o[:, N:] == 5).all()


def test_gradient_with_respect_to_the_input_is_the_operator_itself(ops):
    T, N, D, R, n = 333, 520, 264, 20, 6
    X, W, A, B, ids, s = make(T, N, D, R, n, "mixed")
    dY = torch.randn(T, N, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    dX = ops.gemm_bf16_lora(dY, W, B, A, ids, s, b_is_nk=False)          # W is [N, D]: the [K, N] layout of this product
    within(dX, *exact(dY, W, B, A, ids, s, False, False), "dX")
    # against the derivative of sum(dY * Y) by autograd in 64 bits
    x = X.double().requires_grad_()
    sel = select((x @ A.double().flatten(0, 1).T).view(T, n, R), ids, s.double(), n)
    ((x @ W.double().T + sel @ B.double().flatten(0, 1)) * dY.double()).sum().backward()
    within(dX, x.grad, exact(dY, W, B, A, ids, s, False, False)[1], "dX")


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T,N,D,R,n,order", [
    (1, 8, 8, 1, 1, "one"), (3, 264, 136, 16, 4, "mixed"), (31, 128, 256, 8, 40, "mixed"), (64, 72, 1032, 17, 3, "sorted"), (257, 256, 128, 33, 5, "mixed"),
    (700, 520, 264, 64, 9, "mixed"), (1025, 136, 128, 100, 2, "sorted"), (2000, 256, 512, 128, 3, "one"), (3000, 264, 200, 16, 100, "mixed"),
    (100, 128, 128, 16, 5, "none"), (6000, 64, 64, 16, 1, "one"),
])
def test_adapter_gradients(ops, T, N, D, R, n, order, f32):
    X, W, A, B, ids, s = make(T, N, D, R, n, order, seed=T)
    dY = torch.randn(T, N, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    dt = torch.float32 if f32 else torch.bfloat16
    dA, dB = ops.gemm_bf16_lora_grad(X, dY, A, B, ids, s, out_dtype=dt)
    (gA, tA), (gB, tB) = exact_grad(X, dY, A, B, ids, s, f32)
    within(dA, gA, tA, "dA")
    within(dB, gB, tB, "dB")
    gone = [a for a in range(n) if not (ids == a).any()]
    assert all((dA[a] == 0).all() and (dB[a] == 0).all() for a in gone)
    again = ops.gemm_bf16_lora_grad(X, dY, A, B, ids, s, out_dtype=dt)
    assert torch.equal(dA, again[0]) and torch.equal(dB, again[1])


def test_gradients_keep_requests_apart(ops):
    T, N, D, R, n = 400, 264, 200, 16, 6
    X, W, A, B, ids, s = make(T, N, D, R, n, "mixed")
    dY = torch.randn(T, N, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    want = ops.gemm_bf16_lora_grad(X, dY, A, B, ids, s)
    X2, dY2, A2, B2, i2 = X.clone(), dY.clone(), A.clone(), B.clone(), ids.clone()
    t = int((ids == 2).nonzero()[0])
    X2[t] = NAN
    u = int((ids == 4).nonzero()[0])
    dY2[u] = float("inf")
    B2[1] = NAN
    off = (ids < 0).nonzero()[:, 0]
    X2[off], dY2[off] = NAN, NAN               # rows without an adapter
    i2[off[0]], i2[off[1]] = n, 2 ** 31 - 1    # ids without an adapter
    got = ops.gemm_bf16_lora_grad(X2, dY2, A2, B2, i2, s)
    for a in (0, 3, 5):
        assert torch.equal(got[0][a], want[0][a]) and torch.equal(got[1][a], want[1][a])
    assert got[0][1].isnan().all() and torch.equal(got[1][1], want[1][1])   # B_1 enters dA_1 only
    assert got[0][2].isnan().any() and not got[1][4].isfinite().all()


def test_gradients_against_differences(ops):
    """f = sum(dY * Y) is bilinear in A and B: a central difference along one of them is exact but for the rounding of the
    values of f, so it is taken on FP32 outputs, along directions bf16 holds exactly."""
    T, N, D, R, n = 90, 128, 64, 8, 3
    X, W, A, B, ids, s = make(T, N, D, R, n, "mixed")
    A, B = (A.float() * 256).round().div(256).bfloat16(), (B.float() * 64).round().div(64).bfloat16()
    dY = torch.randn(T, N, generator=torch.Generator().manual_seed(5)).bfloat16().cuda()
    dA, dB = ops.gemm_bf16_lora_grad(X, dY, A, B, ids, s, out_dtype=torch.float32)
    (_, tA), (_, tB) = exact_grad(X, dY, A, B, ids, s, True)
    h = 2.0 ** -4
    g = torch.Generator().manual_seed(3)
    for base, grad, tol, put in ((A, dA, tA, lambda M: (M, B)), (B, dB, tB, lambda M: (A, M))):
        d = (torch.randint(-1, 2, base.shape, generator=g)).cuda().double()
        plus, minus = (base.double() + h * d).bfloat16(), (base.double() - h * d).bfloat16()
        d = (plus.double() - minus.double()) / (2 * h)
        f, noise = [], 0.0
        for M in (plus, minus):
            a, b = put(M)
            y = ops.gemm_bf16_lora(X, W, a, b, ids, s, b_is_nk=True, out_dtype=torch.float32)
            f.append((y.double() * dY.double()).sum())
            noise += (exact(X, W, a, b, ids, s, True, True)[1] * dY.double().abs()).sum()
        bound = noise / (2 * h) + (tol * d.abs()).sum()
        got, want = (f[0] - f[1]) / (2 * h), (grad.double() * d).sum()
        assert abs(got - want) <= bound
        assert bound < 0.05 * (grad.double() * d).abs().sum()


def test_no_tokens(ops):
    X, W, A, B, ids, s = make(4, 64, 64, 8, 2)
    y = ops.gemm_bf16_lora(X[:0], W, A, B, ids[:0], s, b_is_nk=True)
    assert y.shape == (0, 64)
    dA, dB = ops.gemm_bf16_lora_grad(X[:0], torch.zeros(0, 64, device="cuda").bfloat16(), A, B, ids[:0], s)
    assert (dA == 0).all() and (dB == 0).all()


def test_offsets_beyond_32_bits(ops):
    # a stack of adapters of more than 2^31 elements; the last one is used
    n, R, D, N = 4200, 64, 8192, 64
    A = torch.zeros(n, R, D, device="cuda", dtype=torch.bfloat16)
    B = torch.zeros(n, R, N, device="cuda", dtype=torch.bfloat16)
    X, W, a, b, ids, _ = make(20, N, D, R, 1, "one")
    A[-1], B[-1] = a[0], b[0]
    got = ops.gemm_bf16_lora(X, W, A, B, ids + (n - 1), b_is_nk=True)
    assert torch.equal(got, ops.gemm_bf16_lora(X, W, a, b, ids, b_is_nk=True))


def test_captured_graphs_that_replay_at_once(ops):
    """Two graphs, each with scratch of its own, replayed on two streams with new inputs."""
    def step(X, W, A, B, ids, s, dY):
        return (ops.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=True), *ops.gemm_bf16_lora_grad(X, dY, A, B, ids, s))

    states = []
    for seed, (T, N, D, R, n) in enumerate([(40, 512, 4096, 16, 8), (500, 264, 256, 32, 5)]):
        state = (*make(T, N, D, R, n, "mixed", seed=seed), torch.randn(T, N).bfloat16().cuda())
        step(*state)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*state)
        state[0].copy_(torch.randn(T, D).bfloat16())
        state[4].copy_(torch.randint(-1, n, (T,)).int())
        states.append((state, g, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for _, g, _, st in states:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for state, _, out, _ in states:
        assert all(torch.equal(p, q) for p, q in zip(step(*state), out))
    ops.check_status()


def test_refusals_of_the_python_operator(ops):
    X, W, A, B, ids, s = make(8, 128, 64, 8, 2)
    call = lambda **kw: ops.gemm_bf16_lora(**{**dict(X=X, W=W, A=A, B=B, ids=ids, scales=s, b_is_nk=True), **kw})  # noqa: E731
    for kw in (dict(ids=ids.long()), dict(ids=ids[:4]), dict(ids=ids.cpu()), dict(ids=torch.stack([ids, ids], 1)[:, 0]), dict(scales=s.double()),
               dict(scales=s[:1]), dict(A=A[:1]), dict(A=A[:, :4]), dict(B=B[..., :64]), dict(W=W[:, :32]), dict(X=X.float()),
               dict(A=A.transpose(1, 2).contiguous().transpose(1, 2)), dict(out=torch.empty(8, 128, device="cuda")),
               dict(out_dtype=torch.float16)):
        with pytest.raises(ValueError):
            call(**kw)
    from gemm_b200 import GemmB200Error
    with pytest.raises(GemmB200Error):      # adapters that overlap
        call(A=A[:1].expand(2, 8, 64))
    with pytest.raises(GemmB200Error):
        call(A=torch.zeros(2, 129, 64, device="cuda").bfloat16(), B=torch.zeros(2, 129, 128, device="cuda").bfloat16())
    with pytest.raises(ValueError):
        ops.gemm_bf16_lora_grad(X, X, A, B, ids, s)
