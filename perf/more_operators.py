"""Performance cases of what a training step has behind the block operators: ``grouped_gated_product`` (the gated
feed-forward layer of experts or species), ``linear_cross_entropy`` (the loss over a large table without its logits) and
``clip_gradient_norm`` (the norm of all gradients together), through ``mops_b200.torch``, with gradients taken by autograd.

A case is one operator with its sizes, the scalar type and what one pass does: ``"fwd"`` (inference, scoring) or ``"train"`` (forward
and backward). ``own`` selects the framework's kernels; without it the same values come from elementary
torch operations in 32 bits.

Values: groups take rows in proportion to exp(skew * normal), so that some are several times the mean and, where there are
many, some are empty; operands have unit scale and matrices 1/sqrt(K). Targets follow a Zipf-like law, as words do, and some rows
have none (padding, prompts). Gradients of different tensors differ by orders of magnitude.
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# A drawn case has at most so many values in one operand, and so much work in one pass.
MOST_VALUES = 1.3e8
MOST_FLOPS = 8e11
MOST_LOGITS = 8e8
IGNORED = -1


def listed():
    return [
        # a few tokens in flight, each at another expert: the matrices are all that is moved
        dict(name="gated_decode", op="gated", do="fwd", dtype="bf16", R=16, G=32, K=2048, N=1024, skew=0.5, activation="silu"),
        # a prompt through the experts' first layer
        dict(name="gated_prefill", op="gated", do="fwd", dtype="bf16", R=8192, G=16, K=2048, N=1280, skew=0.5, activation="silu"),
        # a training step of it
        dict(name="gated_train", op="gated", do="train", dtype="bf16", R=16384, G=8, K=2048, N=2048, skew=0.5, activation="silu"),
        # a gated layer for each species of atom, in single precision
        dict(name="gated_train_species_f32", op="gated", do="train", dtype="f32", R=100003, G=20, K=128, N=128, skew=1.5, activation="gelu"),
        # odd widths, whose rows start anywhere
        dict(name="gated_train_odd", op="gated", do="train", dtype="f16", R=3001, G=7, K=509, N=387, skew=1.0, activation="gelu"),
        # how likely a few tokens were: the table is all that is moved
        dict(name="loss_score", op="loss", do="fwd", dtype="bf16", R=8, V=50021, C=1024, kept=1.0, weights="mean"),
        # how likely a long text is
        dict(name="loss_text", op="loss", do="fwd", dtype="bf16", R=16384, V=50021, C=1024, kept=0.95, weights="mean"),
        # a training step over words
        dict(name="loss_train_words", op="loss", do="train", dtype="bf16", R=8192, V=100003, C=1024, kept=0.95, weights="mean"),
        # a training step on answers alone (their prompts have no targets), rows weighted, odd widths
        dict(name="loss_train_odd", op="loss", do="train", dtype="f16", R=1537, V=32003, C=771, kept=0.5, weights="rows"),
        # the masked atoms of structures guessed, in single precision
        dict(name="loss_train_f32", op="loss", do="train", dtype="f32", R=4099, V=8009, C=512, kept=0.9, weights="mean"),
        # the gradients of a small model: two dozen tensors, some of a few hundred values
        dict(name="clip_small", op="clip", dtype="f32", tensors=24, width=256, clipped=True),
        # those of a large one, in halves, its norms' weights in single precision
        dict(name="clip_model", op="clip", dtype="bf16", tensors=60, width=2560, clipped=True),
    ]


def _between(rng, low, high):
    """A whole number, spread evenly over the logarithm of the range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["gated", "gated", "loss", "loss", "clip"])
    do = rng.choice(["fwd", "train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    # (in 32 bits the floor is several times higher)
    flops = MOST_FLOPS / (6 if dtype == "f32" else 1) / (3 if do == "train" else 1)
    if op == "clip":
        return dict(op=op, dtype=dtype, tensors=_between(rng, 1, 60), width=_between(rng, 16, 1600), clipped=rng.random() < 0.7)
    if op == "gated":
        K, N = _between(rng, 16, 4096), _between(rng, 16, 2048)
        if rng.random() < 0.6:  # widths of models are mostly multiples of a few elements
            K, N = -(-K // 16) * 16, -(-N // 16) * 16
        G = _between(rng, 1, max(1, min(64, int(MOST_VALUES / (2 * K * N)))))
        R = _between(rng, 1, max(1, min(100003, int(flops / (4 * K * N)), int(MOST_VALUES / max(K, 2 * N)))))
        return dict(op=op, do=do, dtype=dtype, R=R, G=G, K=K, N=N, skew=round(rng.uniform(0.0, 1.5), 2),
                    activation=rng.choice(["silu", "gelu"]))
    C = _between(rng, 16, 4096)
    if rng.random() < 0.6:
        C = -(-C // 16) * 16
    V = _between(rng, 2, min(131072, int(MOST_VALUES / C)))
    R = _between(rng, 1, max(1, min(65536, int(MOST_LOGITS / V), int(flops / (2 * V * C)), int(MOST_VALUES / C))))
    return dict(op=op, do=do, dtype=dtype, R=R, V=V, C=C, kept=round(rng.uniform(0.3, 1.0), 2),
                weights=rng.choice(["mean", "rows"]))


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _shapes(case):
    """The tensors of a model, layer by layer: matrices of a block, then two vectors of its norms."""
    C = case["width"]
    kinds = [(C, C), (C, 2 * C), (2 * C, C), (C, C + C // 2 + 1), (C,), (C,)]
    return [kinds[i % len(kinds)] for i in range(case["tensors"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPE[case["dtype"]]
    s = dict(op=case["op"], do=case.get("do"))
    if case["op"] == "gated":
        R, G, K, N = case["R"], case["G"], case["K"], case["N"]
        share = torch.softmax(case["skew"] * torch.randn(G, generator=gen, device="cuda", dtype=torch.float64), 0)
        group = torch.multinomial(share, R, replacement=True, generator=gen)
        rows = torch.bincount(group, minlength=G)
        s["offsets"] = torch.cat([rows.new_zeros(1), rows.cumsum(0)]).to(torch.int32)
        s["longest"] = int(rows.max())  # the capacity that a program pads to
        s["activation"] = case["activation"]
        s["A"] = _normal(gen, (R, K), dtype)
        s["W"] = _normal(gen, (G, K, 2 * N), dtype, K ** -0.5)
        if case["do"] == "train":
            s["grad"] = _normal(gen, (R, N), dtype)
            s["A"].requires_grad_(True)
            s["W"].requires_grad_(True)
    elif case["op"] == "loss":
        R, V, C = case["R"], case["V"], case["C"]
        s["A"] = _normal(gen, (R, C), dtype)
        s["W"] = _normal(gen, (V, C), dtype, C ** -0.5)
        s["scale"] = 1.25
        # ranks with density ~ 1 / rank, on rows of the table in no particular order
        rank = (V + 1.0) ** torch.rand(R, generator=gen, device="cuda", dtype=torch.float64) - 1.0
        order = torch.randperm(V, generator=gen, device="cuda")
        keep = torch.rand(R, generator=gen, device="cuda") < case["kept"]
        keep[0] = True
        s["targets"] = torch.where(keep, order[rank.long().clamp(0, V - 1)], IGNORED).to(torch.int32)
        if case["do"] == "train":
            weight = keep.float()
            if case["weights"] == "rows":
                weight = weight * (0.5 + torch.rand(R, generator=gen, device="cuda"))
            s["grad_loss"] = weight / weight.sum()  # of the (weighted) mean
            s["grad_log_sum"] = 2e-3 * s["grad_loss"]  # of a small penalty on large sums
            s["A"].requires_grad_(True)
            s["W"].requires_grad_(True)
    else:
        size = torch.exp(0.7 * torch.randn(case["tensors"], generator=gen, device="cuda"))
        s["gradients"] = [(torch.randn(shape, generator=gen, device="cuda") * (1e-3 * size[i])).to(dtype if len(shape) > 1 else torch.float32)
                          for i, shape in enumerate(_shapes(case))]
        values = sum(g.numel() for g in s["gradients"])
        s["max_norm"] = 1e-3 * math.sqrt(values) * (0.25 if case["clipped"] else 25.0)
    return s


# ------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return {"gated": _own_gated, "loss": _own_loss, "clip": _own_clip}[state["op"]](state)
    with torch.no_grad():
        return {"gated": _plain_gated, "loss": _plain_loss, "clip": _plain_clip}[state["op"]](state)


def _own_gated(s):
    import mops_b200.torch as mt
    output = mt.grouped_gated_product(s["A"], s["W"], s["offsets"], s["activation"])
    if s["do"] == "fwd":
        return output
    return output.detach(), *torch.autograd.grad(output, [s["A"], s["W"]], s["grad"])


def _own_loss(s):
    import mops_b200.torch as mt
    loss, log_sum = mt.linear_cross_entropy(s["A"], s["W"], s["targets"], s["scale"], IGNORED)
    if s["do"] == "fwd":
        return loss, log_sum
    return loss.detach(), log_sum.detach(), *torch.autograd.grad([loss, log_sum], [s["A"], s["W"]], [s["grad_loss"], s["grad_log_sum"]])


def _own_clip(s):
    import mops_b200.torch as mt
    norm, clipped = mt.clip_gradient_norm(s["gradients"], s["max_norm"])
    return norm, *clipped


def _plain_gated(s):
    # every group padded to the longest one, then batched products
    A, W, offsets = s["A"], s["W"], s["offsets"].long()
    row = torch.arange(A.shape[0], device=A.device)
    group = torch.searchsorted(offsets, row, right=True) - 1
    within = row - offsets[group]
    at = offsets[:-1, None] + torch.arange(s["longest"], device=A.device)
    inside = (at < offsets[1:, None])[..., None]
    at = at.clamp(max=A.shape[0] - 1)
    padded, W32 = torch.where(inside, A[at].float(), 0.0), W.float()
    u, v = torch.bmm(padded, W32).chunk(2, dim=2)
    if s["activation"] == "silu":
        z = torch.sigmoid(u)
        slope = z * (1 + u * (1 - z))
    else:
        z = 0.5 * torch.erfc(-u * math.sqrt(0.5))
        slope = z + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    output = (u * z * v)[group, within].to(A.dtype)
    if s["do"] == "fwd":
        return output
    grad = torch.where(inside, s["grad"][at].float(), 0.0)
    grad_uv = torch.cat([grad * v * slope, grad * u * z], dim=2)
    grad_A = torch.bmm(grad_uv, W32.transpose(1, 2))[group, within].to(A.dtype)
    return output, grad_A, torch.bmm(padded.transpose(1, 2), grad_uv).to(W.dtype)


def _plain_loss(s):
    A, W, targets = s["A"], s["W"], s["targets"].long()
    keep = targets != IGNORED
    at = torch.where(keep, targets, 0)[:, None]
    A32, W32 = A.float(), W.float()
    x = s["scale"] * (A32 @ W32.T)
    top = x.amax(1)
    log_sum = top + torch.log(torch.exp(x - top[:, None]).sum(1))
    loss = torch.where(keep, log_sum - x.gather(1, at)[:, 0], 0.0)
    if s["do"] == "fwd":
        return loss, torch.where(keep, log_sum, 0.0)
    grad_loss, grad_log_sum = (torch.where(keep, s[g], 0.0)[:, None] for g in ("grad_loss", "grad_log_sum"))
    dx = torch.exp(x - log_sum[:, None]) * (grad_loss + grad_log_sum)
    dx.scatter_add_(1, at, -grad_loss)
    return loss, torch.where(keep, log_sum, 0.0), (s["scale"] * (dx @ W32)).to(A.dtype), (s["scale"] * (dx.T @ A32)).to(W.dtype)


def _plain_clip(s):
    gradients = s["gradients"]
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in gradients]).sum().sqrt()
    factor = (s["max_norm"] / norm).clamp(max=1.0).float()
    return norm.float(), *[(g.float() * factor).to(g.dtype) for g in gradients]


# ------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"gated": _exact_gated, "loss": _exact_loss, "clip": _exact_clip}[case["op"]](s)


def _exact_gated(s):
    # group by group, the gradients by differentiating the definition
    A, W = s["A"].detach().double(), s["W"].detach().double()
    bounds = s["offsets"].tolist()
    N = W.shape[2] // 2
    output, grad_A, grad_W = A.new_zeros((A.shape[0], N)), torch.zeros_like(A), torch.zeros_like(W)
    for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo == hi:
            continue
        with torch.enable_grad():
            a, w = A[lo:hi].clone().requires_grad_(True), W[g].clone().requires_grad_(True)
            u = a @ w[:, :N]
            f = u / (1 + (-u).exp()) if s["activation"] == "silu" else u * (1 + torch.erf(u / math.sqrt(2))) / 2
            h = f * (a @ w[:, N:])
            if s["do"] == "train":
                grad_A[lo:hi], grad_W[g] = torch.autograd.grad(h, [a, w], s["grad"][lo:hi].double())
        output[lo:hi] = h.detach()
    return output if s["do"] == "fwd" else (output, grad_A, grad_W)


def _exact_loss(s):
    # some rows at a time, the gradients by differentiating the definition
    A, W = s["A"].detach().double(), s["W"].detach().double().requires_grad_(True)
    targets, R = s["targets"].long(), s["A"].shape[0]
    loss, log_sum, grad_A, grad_W = A.new_zeros(R), A.new_zeros(R), torch.zeros_like(A), torch.zeros_like(W)
    kept = (targets != IGNORED).nonzero()[:, 0]
    for rows in kept.split(max(1, int(1e8) // W.shape[0])):
        with torch.enable_grad():
            a = A[rows].requires_grad_(True)
            x = torch.nn.functional.linear(a, W) * s["scale"]
            lse = torch.logsumexp(x, 1)
            ce = lse - x[torch.arange(rows.numel(), device=x.device), targets[rows]]
            if s["do"] == "train":
                grad_A[rows], more = torch.autograd.grad([ce, lse], [a, W], [s["grad_loss"][rows].double(), s["grad_log_sum"][rows].double()])
                grad_W += more
        loss[rows], log_sum[rows] = ce.detach(), lse.detach()
    return (loss, log_sum) if s["do"] == "fwd" else (loss, log_sum, grad_A, grad_W.detach())


def _exact_clip(s):
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in s["gradients"]))
    factor = min(1.0, s["max_norm"] / norm)
    return torch.tensor(norm, dtype=torch.float64, device="cuda"), *[g.double() * factor for g in s["gradients"]]


# ------------------------------------------------------------------------- what it costs
def work(case):
    """Bytes: every input read once (of the matrices, those of groups that have rows) and every output written once."""
    size, train = BYTES[case["dtype"]], case.get("do") == "train"
    if case["op"] == "gated":
        R, G, K, N = case["R"], case["G"], case["K"], case["N"]
        move = size * (R * K + min(G, R) * K * 2 * N + R * N) + 4 * (G + 1)
        more = size * (R * N + R * K + G * K * 2 * N) if train else 0
        return {"bytes": move + more, "flops": 4 * R * K * N * (3 if train else 1)}
    if case["op"] == "loss":
        # rows without a target need nothing but their results
        R, V, C = case["R"], case["V"], case["C"]
        kept = max(1, round(R * case["kept"]))
        move = size * (kept * C + V * C) + 4 * R + 8 * R
        more = size * (R * C + V * C) + 8 * R if train else 0
        return {"bytes": move + more, "flops": 2 * kept * V * C * (3 if train else 1)}
    shapes = _shapes(case)
    move = sum(math.prod(shape) * (size if len(shape) > 1 else 4) for shape in shapes)
    return {"bytes": 2 * move + 4, "flops": 3 * sum(math.prod(shape) for shape in shapes)}
