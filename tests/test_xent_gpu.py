"""Softmax cross entropy over a vocabulary projection and its gradient, against the definition in 64 bits.

Tolerances are bounds, element by element.  With u = 2^-24 and a bf16 half step of 2^-8:
  a logit sums D exact products in FP32, in an order and with alignment of the hardware's own: off by at most
  2 (D + 1) u sum |x w| =: ez;
  log-sum-exp: moves by at most max ez, plus the hardware's exponential (2^-21 relative, with its argument's
  rounding (|z| + |lse|) 2 u), plus a few hundred additions (2^-15 covers 512 u);
  d: relative error e = ez(z) + ez(lse) + the above, then one rounding to bf16; dX and dW sum |d| |W| resp. |d| |X| with
  those errors, in FP32, and round to bf16 once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U, HALF = 2.0 ** -24, 2.0 ** -8


def make(T, V, D, seed=0, pad=True, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    X = torch.randn(T, D, generator=g).bfloat16()
    W = (torch.randn(V, D, generator=g) * scale / D ** 0.5).bfloat16()
    lab = torch.randint(0, V, (T,), generator=g)
    lab[0] = V - 1
    if T > 2:
        lab[1] = 0
    if pad and T > 3:
        lab[2::5] = -100
    gl = torch.rand(T, generator=g) - 0.25
    gz = torch.randn(T, generator=g) * 0.1
    return X.cuda(), W.cuda(), lab.cuda(), gl.cuda(), gz.cuda()


def exact(X, W, lab, gl, gz=None):
    """loss, lse, dX, dW in 64 bits, and the bounds on each."""
    x, w = X.double(), W.double()
    D, V = x.shape[1], w.shape[0]
    z = x @ w.T
    lse = torch.logsumexp(z, 1)
    live = lab >= 0
    at = lab.clamp(min=0, max=V - 1)[:, None]
    loss = torch.where(live, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse))
    ez = 2 * (D + 1) * U * (x.abs() @ w.abs().T)
    e_lse = ez.amax(1) + 2.0 ** -21 + 2.0 ** -15 * 1.0 + 2 * U * (z.abs().amax(1) + lse.abs())
    e_loss = e_lse + ez.gather(1, at)[:, 0] + U * loss.abs()
    b = torch.where(live, gl.double(), torch.zeros_like(lse))
    a = b + (gz.double() if gz is not None else 0)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(z).scatter_(1, at, 1.0) * b[:, None]
    d = a[:, None] * p - hot
    rel = ez + (e_lse + 2.0 ** -21 + 4 * U * (lse.abs() + z.abs().amax(1)))[:, None]
    ed = (a[:, None] * p).abs() * rel + (d.abs() + U) * HALF
    dX, dW = d @ w, d.T @ x
    eX = ed @ w.abs() + 2 * (V + 1) * U * (d.abs() @ w.abs()) + HALF * dX.abs()
    eW = ed.T @ x.abs() + 2 * (x.shape[0] + 1) * U * (d.abs().T @ x.abs()) + HALF * dW.abs()
    return (loss, lse, dX, dW), (e_loss, e_lse, 1.02 * eX + 1e-30, 1.02 * eW + 1e-30)


def within(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got.double() - want).abs() / tol).max():.3g} x its bound"


def check(ops, X, W, lab, gl, gz=None):
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    dX, dW = ops.gemm_bf16_xent_grad(X, W, lab, lse, gl, gz)
    ops.check_status()
    want, tol = exact(X, W, lab, gl, gz)
    for got, w, t, what in zip((loss, lse, dX, dW), want, tol, ("loss", "lse", "dX", "dW")):
        within(got, w, t, what)
    return loss, lse, dX, dW


@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (1, 1000, 64), (3, 257, 72), (127, 255, 8), (128, 256, 64), (129, 300, 136), (257, 513, 512),
                                   (64, 5000, 1024), (300, 1001, 200), (1000, 5003, 256), (2, 20011, 2048)])
def test_loss_and_gradient(ops, T, V, D):
    check(ops, *make(T, V, D, seed=T + V))


@pytest.mark.parametrize("T", [16, 31, 32, 33, 64, 65, 128, 129])
def test_around_the_row_counts_where_the_kernels_change(ops, T):
    """32, 64, 128 rows: the box of X; up to 64 rows: d in two bf16 summands; above 128: CTA pairs."""
    check(ops, *make(T, 2050, 264, seed=T))


def test_few_rows_keep_more_of_d_than_one_bf16_value(ops):
    # one row: with a single rounding of the label's entry dX could be off by 2^-8 of itself, now only by its own rounding
    for seed in range(8):
        X, W, lab, gl, _ = make(1, 3000, 256, seed=seed)
        gl = gl.abs() + 0.1
        _, lse = ops.gemm_bf16_xent(X, W, lab)
        dX, dW = ops.gemm_bf16_xent_grad(X, W, lab, lse, gl)
        want, _ = exact(X, W, lab, gl)
        for got, w in ((dX, want[2]), (dW, want[3])):
            off = (got.double() - w).abs()
            # its own half step, two summands of d (2^-16) and the logits' and log-sum-exp's FP32 errors (below 2^-14)
            assert (off <= HALF * w.abs() + 2.0 ** -13 * w.abs().max()).all()


def test_gradient_through_the_log_sum_exp(ops):
    check(ops, *make(200, 777, 128)[:4], make(200, 777, 128)[4])


def test_vocabulary_in_several_pieces(ops):
    # 2 T V bytes of d are over the size of one piece: dX is summed over pieces, the last of them shorter
    X, W, lab, gl, gz = make(4100, 70001, 64)
    check(ops, X, W, lab, gl / 4100, None)


def test_long_hidden_size_takes_the_run_time_schedule(ops):
    check(ops, *make(700, 9000, 6144, scale=1.0)[:4])


def test_few_tokens_long_vocabulary_split_over_k(ops):
    # dX has few tiles and a long K (the vocabulary); dW of a small vocabulary has few tiles and many tokens
    check(ops, *make(40, 40000, 256)[:4])
    check(ops, *make(9000, 300, 128)[:4])


def test_forward_takes_a_hidden_size_of_any_parity(ops):
    X, W, lab, gl, _ = make(33, 400, 24)
    X, W = X[:, :21], W[:, :21]
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    want, tol = exact(X, W, lab, gl)
    within(loss, want[0], tol[0], "loss")
    within(lse, want[1], tol[1], "lse")


def test_strided_operands_and_outputs_leave_their_neighbours_alone(ops):
    T, V, D = 130, 515, 72
    X, W, lab, gl, gz = make(T, V, D)
    Xw, Ww = torch.full((T, D + 8), 7.0, device="cuda").bfloat16(), torch.full((V, D + 24), -3.0, device="cuda").bfloat16()
    Xw[:, :D], Ww[:, 8:8 + D] = X, W
    plain = check(ops, X, W, lab, gl, gz)
    g2 = torch.stack([gl, torch.full_like(gl, 9.0)], 1)
    oX, oW = torch.full((T + 3, D + 16), 5.0, device="cuda").bfloat16(), torch.full((V + 2, D + 8), 5.0, device="cuda").bfloat16()
    loss, lse = ops.gemm_bf16_xent(Xw[:, :D], Ww[:, 8:8 + D], lab)
    dX, dW = ops.gemm_bf16_xent_grad(Xw[:, :D], Ww[:, 8:8 + D], lab, lse, g2[:, 0], gz, out=(oX[:T, :D], oW[:V, :D]))
    for got, want in zip((loss, lse, dX, dW), plain):
        assert torch.equal(got, want)
    for o, r in ((oX, T), (oW, V)):
        assert (o[r:] == 5).all() and (o[:, D:] == 5).all()


def test_expanded_scalar_gradient(ops):
    X, W, lab, gl, _ = make(100, 300, 64)
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    one = torch.full((), 0.01, device="cuda")
    a = ops.gemm_bf16_xent_grad(X, W, lab, lse, one.expand(100))
    b = ops.gemm_bf16_xent_grad(X, W, lab, lse, torch.full((100,), 0.01, device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_padding_rows_hold_anything(ops):
    X, W, lab, gl, _ = make(140, 300, 64)
    pad = lab < 0
    X0, X1, g1 = X.clone(), X.clone(), gl.clone()
    X0[pad] = 0
    X1[pad] = float("nan")
    X1[2] = float("inf")
    g1[pad] = float("nan")            # not read
    loss, lse = ops.gemm_bf16_xent(X1, W, lab)
    assert (loss[pad] == 0).all() and loss.isfinite().all()
    got = ops.gemm_bf16_xent_grad(X1, W, lab, lse, g1)
    loss0, lse0 = ops.gemm_bf16_xent(X0, W, lab)
    want = ops.gemm_bf16_xent_grad(X0, W, lab, lse0, gl)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (got[0][pad] == 0).all()


def test_every_row_padding(ops):
    X, W, lab, gl, _ = make(50, 300, 64)
    lab.fill_(-1)
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    dX, dW = ops.gemm_bf16_xent_grad(X, W, lab, lse, gl)
    assert (loss == 0).all() and (dX == 0).all() and (dW == 0).all()


def test_labels_outside_the_vocabulary(ops):
    X, W, lab, gl, _ = make(40, 300, 64)
    lab[5], lab[6] = 300, 1 << 40
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    bad = torch.tensor([5, 6], device="cuda")
    assert loss[bad].isnan().all() and int(loss.isnan().sum()) == 2 and lse.isfinite().all()
    dX, _ = ops.gemm_bf16_xent_grad(X, W, lab, lse, gl)
    assert dX[bad].isnan().all() and int(dX.isnan().any(1).sum()) == 2


def test_infinite_and_nan_logits_follow_logsumexp(ops):
    V, D = 700, 8
    W = torch.ones(V, D, device="cuda").bfloat16()
    W[:300] = 0.5                     # whole tiles, and part of one, at another height
    X = torch.zeros(6, D, device="cuda").bfloat16()
    X[0, 0] = float("inf")            # every logit +inf
    X[1, 0] = float("-inf")           # every logit -inf
    X[2, 0] = float("nan")
    X[3] = 1.0
    X[4] = -3e4                       # far apart, all negative
    lab = torch.tensor([0, 0, 0, 1, 0, -1], device="cuda")
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    z = X.double() @ W.double().T
    want = torch.logsumexp(z, 1)
    assert lse[0] == float("inf") and lse[1] == float("-inf") and lse[2].isnan()
    torch.testing.assert_close(lse[3:].double(), want[3:], rtol=2.0 ** -19, atol=2.0 ** -15)
    # one vocabulary entry switched off (its logit -inf), and one tile's worth of them
    W2 = W.clone()
    W2[10, 1] = float("-inf")
    W2[256:512, 1] = float("-inf")
    loss, lse = ops.gemm_bf16_xent(X[3:4], W2, lab[3:4])
    z = X[3:4].double() @ W2.double().T
    torch.testing.assert_close(lse.double(), torch.logsumexp(z, 1), rtol=0, atol=2.0 ** -15)
    assert loss.isfinite().all()


def test_large_logits_do_not_overflow(ops):
    X, W, lab, gl, _ = make(130, 700, 64, scale=500.0)
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    want, tol = exact(X, W, lab, gl)
    within(lse, want[1], tol[1], "lse")
    within(loss, want[0], tol[0], "loss")
    dX, dW = ops.gemm_bf16_xent_grad(X, W, lab, lse, gl)
    assert dX.isfinite().all() and dW.isfinite().all()


def test_no_tokens(ops):
    X, W = torch.zeros(0, 64, device="cuda").bfloat16(), torch.ones(300, 64, device="cuda").bfloat16()
    e = torch.zeros(0, device="cuda")
    loss, lse = ops.gemm_bf16_xent(X, W, e.long())
    assert loss.shape == (0,) and lse.shape == (0,)
    dX, dW = ops.gemm_bf16_xent_grad(X, W, e.long(), lse, e)
    assert dX.shape == (0, 64) and (dW == 0).all()


def test_gradient_against_differences(ops):
    """Along directions U that bf16 holds exactly: f(h) = sum g loss(X + h U) has |f'''| <= sum |g| (2 S)^3 with S the largest
    |slope| of a logit, so the central difference is off by h^2 / 6 of that, and by the losses' errors / h."""
    T, V, D = 37, 301, 64
    X, W, lab, gl, _ = make(T, V, D)
    X, W = (X.float() * 16).round().div(16).bfloat16(), (W.float() * 64).round().div(64).bfloat16()   # room for the steps
    h = 2.0 ** -5
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    dX, dW = ops.gemm_bf16_xent_grad(X, W, lab, lse, gl)
    _, tol = exact(X, W, lab, gl)
    g = torch.Generator().manual_seed(3)
    live = (lab >= 0).double()
    for which in ("X", "W"):
        base, grad, etol = (X, dX, tol[2]) if which == "X" else (W, dW, tol[3])
        Udir = (torch.randint(0, 2, base.shape, generator=g) * 2 - 1).cuda().double() * (torch.rand(base.shape, generator=g) < 0.05).cuda()
        plus, minus = (base.double() + h * Udir).bfloat16(), (base.double() - h * Udir).bfloat16()
        Udir = (plus.double() - minus.double()) / (2 * h)      # the step that was taken
        args = [(plus, W), (minus, W)] if which == "X" else [(X, plus), (X, minus)]
        f = [(ops.gemm_bf16_xent(a, b, lab)[0].double() * gl.double() * live).sum() for a, b in args]
        S = (Udir @ W.double().T if which == "X" else X.double() @ Udir.T).abs().amax(1)
        bound = (gl.abs().double() * (2 * S) ** 3).sum() * h * h / 6 + (gl.abs().double() * tol[0]).sum() / h * 2 + (etol * Udir.abs()).sum()
        assert abs((f[0] - f[1]) / (2 * h) - (grad.double() * Udir).sum()) <= bound
        assert bound < 0.5 * (grad.double() * Udir).abs().sum()   # the bound says something


def test_runs_repeat_bit_for_bit(ops):
    X, W, lab, gl, gz = make(600, 3001, 256)
    a = (*ops.gemm_bf16_xent(X, W, lab),)
    a += (*ops.gemm_bf16_xent_grad(X, W, lab, a[1], gl, gz),)
    for _ in range(3):
        b = (*ops.gemm_bf16_xent(X, W, lab),)
        b += (*ops.gemm_bf16_xent_grad(X, W, lab, b[1], gl, gz),)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_graphs_that_replay_at_once(ops):
    """Two graphs, each with scratch of its own, replayed on two streams with new inputs."""
    states, graphs = [], []
    for seed, (T, V, D) in enumerate([(300, 2001, 128), (77, 5000, 256)]):
        X, W, lab, gl, _ = make(T, V, D, seed=seed)
        ops.gemm_bf16_xent_grad(X, W, lab, ops.gemm_bf16_xent(X, W, lab)[1], gl)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            loss, lse = ops.gemm_bf16_xent(X, W, lab)
            dX, dW = ops.gemm_bf16_xent_grad(X, W, lab, lse, gl)
        states.append((X, W, lab, gl, loss, lse, dX, dW))
        graphs.append(g)
    for seed, s in enumerate(states):
        new = make(*s[0].shape[:1], s[1].shape[0], s[0].shape[1], seed=10 + seed)
        for dst, src in zip(s[:4], new):
            dst.copy_(src)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for X, W, lab, gl, loss, lse, dX, dW in states:
        a = ops.gemm_bf16_xent(X, W, lab)
        b = ops.gemm_bf16_xent_grad(X, W, lab, a[1], gl)
        assert all(torch.equal(p, q) for p, q in zip((loss, lse, dX, dW), (*a, *b)))
    ops.check_status()


def test_on_a_stream_of_its_own(ops):
    X, W, lab, gl, _ = make(200, 1000, 128)
    want = check(ops, X, W, lab, gl)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = [(*ops.gemm_bf16_xent(X, W, lab),) for _ in range(20)]
        got = [(*f, *ops.gemm_bf16_xent_grad(X, W, lab, f[1], gl)) for f in got]
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for f in got for p, q in zip(f, want))


def test_refusals_of_the_python_operator(ops):
    X, W, lab, gl, _ = make(8, 100, 64)
    for bad in (lab.int(), lab[:7], lab.cpu(), lab[None]):
        with pytest.raises(ValueError):
            ops.gemm_bf16_xent(X, W, bad)
    with pytest.raises(ValueError):
        ops.gemm_bf16_xent(X.float(), W, lab)
    with pytest.raises(ValueError):
        ops.gemm_bf16_xent(X, W[:, :32], lab)
    with pytest.raises(ValueError):
        ops.gemm_bf16_xent(X, W.t().contiguous().t(), lab)          # W must be row-major
    loss, lse = ops.gemm_bf16_xent(X, W, lab)
    for bad in (gl.double(), gl[:3], gl.sum()):
        with pytest.raises(ValueError):
            ops.gemm_bf16_xent_grad(X, W, lab, lse, bad)
    with pytest.raises(ValueError):
        ops.gemm_bf16_xent_grad(X, W, lab, lse, gl, out=(torch.empty_like(X), torch.empty_like(X)))
    from gemm_b200 import GemmB200Error
    with pytest.raises(GemmB200Error):
        ops.gemm_bf16_xent(X[:, 1:], W[:, 1:], lab)                 # misaligned
    with pytest.raises(GemmB200Error):
        ops.gemm_bf16_xent_grad(X[:, :60], W[:, :60], lab, lse, gl)   # D no multiple of 8
    with pytest.raises(GemmB200Error):
        ops.gemm_bf16_xent(X, W[:0], lab)
