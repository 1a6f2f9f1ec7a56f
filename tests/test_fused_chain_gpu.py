"""The operators as they are used together: a projection with the adapters of several requests, the loss over a
vocabulary projection behind it, and one backward pass through both to the adapters; as torch.library operators; and
from a captured graph that was never run eagerly."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def setup(T=300, D=256, N=512, V=3001, R=16, n=5, seed=0):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn(T, D, generator=g).bfloat16().cuda()
    W = (torch.randn(N, D, generator=g) / D ** 0.5).bfloat16().cuda()
    A = (torch.randn(n, R, D, generator=g) / D ** 0.5).bfloat16().cuda()
    B = (torch.randn(n, R, N, generator=g) / R ** 0.5).bfloat16().cuda()
    H = (torch.randn(V, N, generator=g) / N ** 0.5).bfloat16().cuda()
    ids = torch.randint(-1, n, (T,), generator=g).int().cuda()
    s = (torch.rand(n, generator=g) + 0.5).cuda()
    labels = torch.randint(0, V, (T,), generator=g).cuda()
    labels[::7] = -100
    return X, W, A, B, H, ids, s, labels


def step(ops, X, W, A, B, H, ids, s, labels):
    Y = ops.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=True)
    loss, lse = ops.gemm_bf16_xent(Y, H, labels)
    w = (labels >= 0).float() / labels.numel()
    dY, dH = ops.gemm_bf16_xent_grad(Y, H, labels, lse, w)
    dA, dB = ops.gemm_bf16_lora_grad(X, dY, A, B, ids, s, out_dtype=torch.float32)
    dX = ops.gemm_bf16_lora(dY, W, B, A, ids, s, b_is_nk=False)
    return Y, loss, dY, dH, dA, dB, dX


def test_fine_tuning_step(ops):
    """Against 64 bits from the rounded intermediate results on: each operator sees the bf16 tensor that the one before it
    gave, so each is held to its own bound: relative, a bf16 half step (2^-8) for each rounding on the way (d or V,
    and the result), and FP32 sums."""
    X, W, A, B, H, ids, s, labels = state = setup()
    Y, loss, dY, dH, dA, dB, dX = step(ops, *state)
    ops.check_status()
    n, R, D = A.shape
    T = X.shape[0]

    def rel(got, want):
        return ((got.double() - want).norm() / want.norm()).item()

    mine = (ids[:, None] == torch.arange(n, device=ids.device))[..., None]
    pick = lambda P, M: torch.where(mine, (P.double() @ M.double().flatten(0, 1).T).view(T, n, R) * s.double().view(1, n, 1), 0.0).flatten(1)  # noqa: E731
    assert rel(Y, X.double() @ W.double().T + pick(X, A) @ B.double().flatten(0, 1)) < 2 * 2.0 ** -8
    z = Y.double() @ H.double().T
    live = labels >= 0
    want = torch.where(live, torch.logsumexp(z, 1) - z.gather(1, labels.clamp(min=0)[:, None])[:, 0], 0.0)
    assert rel(loss, want) < 2.0 ** -18
    d = torch.softmax(z, 1)
    d[live.nonzero()[:, 0], labels[live]] -= 1
    d *= (live.double() / T)[:, None]
    assert rel(dY, d @ H.double()) < 2 * 2.0 ** -8 and rel(dH, d.T @ Y.double()) < 2 * 2.0 ** -8
    assert rel(dA, (pick(dY, B).T @ X.double()).view(A.shape)) < 2.0 ** -18
    assert rel(dB, (pick(X, A).T @ dY.double()).view(B.shape)) < 2.0 ** -18
    assert rel(dX, dY.double() @ W.double() + pick(dY, B) @ A.double().flatten(0, 1)) < 2 * 2.0 ** -8


def test_a_step_captured_without_a_first_run(ops):
    states = [setup(seed=3), setup(T=40, D=4096, N=264, V=900, seed=4)]
    graphs = []
    for state in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(ops, *state)
        graphs.append((g, out))
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for state, (_, out) in zip(states, graphs):
        assert all(torch.equal(a, b) for a, b in zip(out, step(ops, *state)))
    ops.check_status()


def test_two_threads_on_two_streams(ops):
    import threading
    states = [setup(seed=5), setup(T=700, D=512, N=264, V=1500, R=40, n=9, seed=6)]
    want = [step(ops, *s) for s in states]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    got[i] = step(ops, *states[i])
            st.synchronize()
        except Exception as e:   # a thread's exception would be lost
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for w, g in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(w, g))
    ops.check_status()


def test_as_torch_library_operators(ops):
    import gemm_b200.torch_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    X, W, A, B, H, ids, s, labels = state = setup()
    lib = torch.ops.gemm_b200
    Y, loss, dY, dH, dA, dB, _ = step(ops, *state)
    w = (labels >= 0).float() / labels.numel()

    def run(X, W, A, B, H, ids, s, labels, w):
        y = lib.gemm_bf16_lora(X, W, A, B, ids, s, b_is_nk=True)
        l, lse = lib.gemm_bf16_xent(y, H, labels)
        dy, dh = lib.gemm_bf16_xent_grad(y, H, labels, lse, w)
        da, db = lib.gemm_bf16_lora_grad(X, dy, A, B, ids, s, out_f32=True)
        return y, l, dy, dh, da, db

    real = run(*state, w)
    assert all(torch.equal(a, b) for a, b in zip(real, (Y, loss, dY, dH, dA, dB)))
    with FakeTensorMode() as mode:
        fake = run(*[mode.from_tensor(t) for t in (*state, w)])
    assert all(f.shape == r.shape and f.dtype == r.dtype for f, r in zip(fake, real))
