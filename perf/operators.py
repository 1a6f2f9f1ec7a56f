"""What is measured of the language-model operators that stand beside the BF16 GEMM.

Four operators, in two pairs:

* ``xent``       softmax cross entropy over a vocabulary projection, ``gemm_bf16_xent``
* ``xent_step``  the same with its gradient, ``gemm_bf16_xent`` and then ``gemm_bf16_xent_grad``
* ``lora``       a projection with the low-rank adapters of many requests beside it, ``gemm_bf16_lora``
* ``lora_grad``  the gradient of those adapters, ``gemm_bf16_lora_grad``

Where ``own`` is false, ``run`` computes them with elementary torch operations in 32 bits."""
import math

import torch

own = False

XENT = dict(op="xent")
STEP = dict(op="xent_step")
LORA = dict(op="lora")
GRAD = dict(op="lora_grad")


def listed():
    return [
        # one position scored against the whole vocabulary: what a server asks for with each token's log-probability
        dict(XENT, name="xent one token", T=1, D=4096, V=131072),
        # an evaluation batch of ragged length over a vocabulary that is no multiple of anything
        dict(XENT, name="xent ragged batch", T=509, D=1024, V=50001),
        # perplexity over a long document
        dict(XENT, name="xent long", T=4096, D=4096, V=131072),
        # a short fine-tuning batch
        dict(STEP, name="step short", T=67, D=2048, V=32001),
        # a training micro-batch
        dict(STEP, name="step training", T=8192, D=4096, V=131072),
        # one request decodes with its adapter, seven others are loaded
        dict(LORA, name="lora one token", T=1, D=4096, N=4096, R=16, adapters=8, requests=1, plain_rows=0, sorted=True, nk=True, f32=False),
        # a decoding batch in arrival order: 32 adapters and a few requests without one
        dict(LORA, name="lora decode", T=48, D=8192, N=8192, R=16, adapters=64, requests=32, plain_rows=5, sorted=False, nk=True, f32=False),
        # prompts and single tokens of 20 requests together, of odd length, FP32 output into a reduction
        dict(LORA, name="lora mixed f32", T=1003, D=4096, N=8192, R=64, adapters=20, requests=20, plain_rows=64, sorted=True, nk=False, f32=True),
        # prompts of 16 requests
        dict(LORA, name="lora prompts", T=8192, D=8192, N=8192, R=16, adapters=16, requests=16, plain_rows=0, sorted=True, nk=True, f32=False),
        # a small batch that trains three adapters
        dict(GRAD, name="lora grad small", T=300, D=2048, N=2048, R=8, adapters=3, requests=3, plain_rows=10, sorted=False, f32=False),
        # a training batch of four adapters, gradients in FP32 for the optimiser
        dict(GRAD, name="lora grad training", T=8192, D=4096, N=8192, R=32, adapters=4, requests=4, plain_rows=0, sorted=True, f32=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _eights(rng, lo, hi):
    return 8 * _log(rng, lo // 8, hi // 8)


def draw(rng):
    op = rng.choice(["xent", "xent_step", "lora", "lora", "lora_grad"])
    T = _log(rng, 1, 8192)
    if op.startswith("xent"):
        return dict(op=op, T=T, D=_eights(rng, 256, 4096), V=_log(rng, 1000, 131072))
    adapters = _log(rng, 1, 64)
    case = dict(op=op, T=T, D=_eights(rng, 512, 8192), N=_eights(rng, 512, 8192), R=_log(rng, 1, 128), adapters=adapters,
                requests=min(T, rng.randint(1, adapters)), plain_rows=0, sorted=rng.random() < 0.6, f32=rng.random() < 0.4)
    if rng.random() < 0.5:
        case["plain_rows"] = rng.randint(0, T - case["requests"])
    if op == "lora":
        case["nk"] = rng.random() < 0.6
    return case


def _normal(gen, shape, std):
    return (torch.randn(shape, generator=gen, device="cuda") * std).bfloat16()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    T, D = case["T"], case["D"]
    s = dict(op=case["op"], X=_normal(gen, (T, D), 1.0))
    if case["op"].startswith("xent"):
        V = case["V"]
        s["W"] = _normal(gen, (V, D), 2.0 / math.sqrt(D))   # logits of standard deviation 2
        labels = torch.randint(0, V, (T,), generator=gen, device="cuda")
        if T > 8:   # padding
            labels = torch.where(torch.rand(T, generator=gen, device="cuda") < 0.1, torch.full_like(labels, -100), labels)
        s["labels"] = labels
        s["grad_loss"] = torch.rand(T, generator=gen, device="cuda") / T   # weighted mean over the batch
        return s
    N, R, n = case["N"], case["R"], case["adapters"]
    # every request has an adapter of its own and at least one row; the rest of the rows go to any of them
    free = torch.randint(0, case["requests"], (T,), generator=gen, device="cuda")
    ids = torch.cat([torch.arange(case["requests"], device="cuda"), free])[:T]
    ids[T - case["plain_rows"]:] = -1   # rows without an adapter
    if case["sorted"]:
        ids = torch.sort(ids)[0]
    else:
        ids = ids[torch.randperm(T, generator=gen, device="cuda")]
    which = torch.randperm(n, generator=gen, device="cuda")
    if case["sorted"]:
        which = torch.sort(which[:case["requests"]])[0]
    s["ids"] = torch.where(ids >= 0, which[ids.clamp(min=0)], ids).int()
    s["A"] = _normal(gen, (n, R, D), 1.0 / math.sqrt(D))
    s["B"] = _normal(gen, (n, R, N), 1.0 / math.sqrt(R))
    s["scales"] = 0.25 + 0.5 * torch.rand(n, generator=gen, device="cuda")
    s["out"] = torch.float32 if case["f32"] else torch.bfloat16
    if case["op"] == "lora":
        s["nk"] = case["nk"]
        s["W"] = _normal(gen, (N, D) if case["nk"] else (D, N), 1.0 / math.sqrt(D))
    else:
        s["dY"] = _normal(gen, (T, N), 1.0 / T)
    return s


def _chosen(products, ids, scales):
    """Of the products with every adapter [T, adapters * R], the row's own, scaled; zero elsewhere."""
    n = scales.numel()
    p = products.view(products.shape[0], n, -1)
    mine = ids.view(-1, 1) == torch.arange(n, device=ids.device)
    return torch.where(mine.unsqueeze(2), p * scales.view(1, n, 1), torch.zeros((), device=p.device)).flatten(1)


def _plain(s):
    X = s["X"].float()
    if s["op"].startswith("xent"):
        W, labels = s["W"].float(), s["labels"]
        logits = X @ W.t()
        top = logits.max(dim=1, keepdim=True).values
        p = torch.exp(logits - top)
        total = p.sum(dim=1, keepdim=True)
        lse = (top + torch.log(total)).squeeze(1)
        live = labels >= 0
        at = labels.clamp(min=0).unsqueeze(1)
        loss = torch.where(live, lse - logits.gather(1, at).squeeze(1), torch.zeros_like(lse))
        if s["op"] == "xent":
            return loss, lse
        g = torch.where(live, s["grad_loss"], torch.zeros_like(lse)).unsqueeze(1)
        p.mul_(g / total)
        p.scatter_add_(1, at, -g)
        return loss, lse, (p @ W).bfloat16(), (p.t() @ X).bfloat16()
    A, B, ids, scales = s["A"].float(), s["B"].float(), s["ids"], s["scales"]
    v = _chosen(X @ A.flatten(0, 1).t(), ids, scales)
    if s["op"] == "lora":
        W = s["W"].float()
        return (X @ (W.t() if s["nk"] else W) + v @ B.flatten(0, 1)).to(s["out"])
    dY = s["dY"].float()
    u = _chosen(dY @ B.flatten(0, 1).t(), ids, scales)
    return (u.t() @ X).view(A.shape).to(s["out"]), (v.t() @ dY).view(B.shape).to(s["out"])


def run(state):
    s = state
    if not own:
        return _plain(s)
    import gemm_b200 as g
    if s["op"].startswith("xent"):
        loss, lse = g.gemm_bf16_xent(s["X"], s["W"], s["labels"])
        if s["op"] == "xent":
            return loss, lse
        dX, dW = g.gemm_bf16_xent_grad(s["X"], s["W"], s["labels"], lse, s["grad_loss"])
        return loss, lse, dX, dW
    if s["op"] == "lora":
        return g.gemm_bf16_lora(s["X"], s["W"], s["A"], s["B"], s["ids"], s["scales"], b_is_nk=s["nk"], out_dtype=s["out"])
    return g.gemm_bf16_lora_grad(s["X"], s["dY"], s["A"], s["B"], s["ids"], s["scales"], out_dtype=s["out"])


def work(case):
    T, D = case["T"], case["D"]
    if case["op"].startswith("xent"):
        V = case["V"]
        once = 2 * (T * D + V * D) + 8 * T + 8 * T   # hidden states and weights; labels; loss and log-sum-exp
        if case["op"] == "xent":
            return {"bytes": once, "flops": 2 * T * V * D}
        return {"bytes": once + 4 * T + 2 * (T * D + V * D), "flops": 6 * T * V * D}
    N, R, out = case["N"], case["R"], 4 if case["f32"] else 2
    rows = T - case["plain_rows"]                     # rows that have an adapter
    low = 2 * case["requests"] * R * (D + N) + 4 * T    # the adapters in use, the rows' choice of them
    if case["op"] == "lora":
        return {"bytes": 2 * (T * D + D * N) + low + out * T * N, "flops": 2 * T * D * N + 2 * rows * R * (D + N)}
    return {"bytes": 2 * rows * (D + N) + low + out * case["adapters"] * R * (D + N), "flops": 4 * rows * R * (D + N)}


def exact(case, seed):
    s = prepare(case, seed)
    X = s["X"].double()
    T = X.shape[0]
    if case["op"].startswith("xent"):
        W, labels = s["W"].double(), s["labels"]
        loss, lse = X.new_zeros(T), X.new_zeros(T)
        step = case["op"] == "xent_step"
        dX, dW = (torch.zeros_like(X), torch.zeros_like(W)) if step else (None, None)
        for a in range(0, T, 1024):
            rows = slice(a, min(T, a + 1024))
            z = torch.mm(X[rows], W.T)
            lse[rows] = torch.logsumexp(z, 1)
            live = (labels[rows] >= 0).nonzero()[:, 0]
            hit = labels[rows][live]
            loss[rows][live] = lse[rows][live] - z[live, hit]
            if step:
                w = torch.zeros(z.shape[0], dtype=torch.float64, device=z.device)
                w[live] = s["grad_loss"][rows][live].double()
                z = torch.softmax(z, 1)
                z[live, hit] -= 1
                z *= w[:, None]
                dX[rows] = torch.mm(z, W)
                dW.addmm_(z.T, X[rows])
        return (loss, lse, dX, dW) if step else (loss, lse)
    A, B = s["A"].double(), s["B"].double()
    ids, scales = s["ids"].tolist(), s["scales"].double()
    member = {}
    for t, i in enumerate(ids):
        member.setdefault(i, []).append(t)
    member.pop(-1, None)
    if case["op"] == "lora":
        y = torch.mm(X, s["W"].double().T if case["nk"] else s["W"].double())
        for i, rows in member.items():
            y[rows] += scales[i] * torch.mm(torch.mm(X[rows], A[i].T), B[i])
        return y
    dY = s["dY"].double()
    dA, dB = torch.zeros_like(A), torch.zeros_like(B)
    for i, rows in member.items():
        dA[i] = scales[i] * torch.mm(torch.mm(dY[rows], B[i].T).T, X[rows])
        dB[i] = scales[i] * torch.mm(torch.mm(X[rows], A[i].T).T, dY[rows])
    return dA, dB
