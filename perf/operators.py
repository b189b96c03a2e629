"""Performance cases of the block operators: ``embedding_lookup``, ``grouped_matrix_product`` and
``gated_residual_norm``, through ``mops_b200.torch``, with gradients taken by autograd.

A case is one operator with its sizes, the scalar type and what one pass does: ``"fwd"``
(inference) or ``"train"`` (forward and backward). ``own`` selects the framework's kernels;
without it the same values come from elementary torch operations in 32 bits.

Values: token ids follow a Zipf-like law, as words do (and as the species of atoms do: a few are most
of them); groups take rows in proportion to exp(skew * normal), so that some are several times the
mean and, where there are many, some are empty; operands have unit scale and matrices 1/sqrt(K).
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}

# A drawn case has at most so many values in one operand, and so much work in one pass.
MOST_VALUES = 1.3e8
MOST_FLOPS = 4e11


def listed():
    return [
        # eight sequences, one token each: nothing but latency
        dict(name="embedding_decode", op="embedding", do="fwd", dtype="bf16", T=8, V=50021, D=1024),
        # a long prompt, or many of them, with a large vocabulary
        dict(name="embedding_prefill", op="embedding", do="fwd", dtype="bf16", T=65536, V=131072, D=2048),
        # a training step over words: most rows of the table get no token, a few get thousands
        dict(name="embedding_train_words", op="embedding", do="train", dtype="bf16", T=16384, V=100003, D=1024),
        # a training step over the atoms of a batch of structures: a handful of rows get everything
        dict(name="embedding_train_species", op="embedding", do="train", dtype="f32", T=200003, V=95, D=256),
        # a few tokens in flight, each at another expert: the matrices are all that is moved
        dict(name="experts_decode", op="grouped", do="fwd", dtype="bf16", R=16, G=32, K=2048, N=1536, skew=0.5),
        # a prompt through the experts
        dict(name="experts_prefill", op="grouped", do="fwd", dtype="bf16", R=8192, G=16, K=2048, N=1536, skew=0.5),
        # a training step of the experts' first product
        dict(name="experts_train", op="grouped", do="train", dtype="bf16", R=16384, G=8, K=2048, N=4096, skew=0.5),
        # a linear map for each species of atom, in single precision
        dict(name="species_train_f32", op="grouped", do="train", dtype="f32", R=100003, G=20, K=128, N=128, skew=1.5),
        # odd widths, whose rows start anywhere
        dict(name="experts_train_odd", op="grouped", do="train", dtype="bf16", R=3001, G=7, K=509, N=771, skew=1.0),
        # one token of four sequences
        dict(name="norm_decode", op="norm", do="fwd", dtype="bf16", R=4, C=4096, gate="full"),
        # a training step of a wide model
        dict(name="norm_train", op="norm", do="train", dtype="bf16", R=16384, C=4096, gate="full"),
        # features of atoms, one gate for each, in single precision, an odd number of rows
        dict(name="norm_train_rows_f32", op="norm", do="train", dtype="f32", R=20011, C=1000, gate="row"),
    ]


def _between(rng, low, high):
    """A whole number, spread evenly over the logarithm of the range."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    op = rng.choice(["embedding", "grouped", "grouped", "norm"])
    do = rng.choice(["fwd", "train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "embedding":
        D = _between(rng, 16, 4096)
        most = int(MOST_VALUES / D)
        return dict(op=op, do=do, dtype=dtype, D=D, T=_between(rng, 1, min(200003, most)),
                    V=_between(rng, 2, min(131072, most)))
    if op == "norm":
        C = _between(rng, 16, 8192)
        return dict(op=op, do=do, dtype=dtype, C=C, R=_between(rng, 1, min(65536, int(6.7e7 / C))),
                    gate=rng.choice(["full", "row", "none"]))
    K, N = _between(rng, 16, 4096), _between(rng, 16, 4096)
    if rng.random() < 0.6:  # widths of models are mostly multiples of a few elements
        K, N = -(-K // 16) * 16, -(-N // 16) * 16
    G = _between(rng, 1, max(1, min(64, int(MOST_VALUES / (K * N)))))
    # (in 32 bits the floor is several times higher)
    flops = MOST_FLOPS / (6 if dtype == "f32" else 1) / (3 if do == "train" else 1)
    R = _between(rng, 1, max(1, min(100003, int(flops / (2 * K * N)), int(MOST_VALUES / max(K, N)))))
    return dict(op=op, do=do, dtype=dtype, R=R, G=G, K=K, N=N, skew=round(rng.uniform(0.0, 1.5), 2))


def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPE[case["dtype"]]
    s = dict(op=case["op"], do=case["do"])
    if case["op"] == "embedding":
        T, V, D = case["T"], case["V"], case["D"]
        s["W"] = _normal(gen, (V, D), dtype, D ** -0.5)
        # ranks with density ~ 1 / rank, on rows of the table in no particular order
        rank = (V + 1.0) ** torch.rand(T, generator=gen, device="cuda", dtype=torch.float64) - 1.0
        order = torch.randperm(V, generator=gen, device="cuda")
        s["indices"] = order[rank.long().clamp(0, V - 1)].to(torch.int32)
        s["scale"] = math.sqrt(D)
        if case["do"] == "train":
            s["grad"] = _normal(gen, (T, D), dtype)
            s["W"].requires_grad_(True)
    elif case["op"] == "grouped":
        R, G, K, N = case["R"], case["G"], case["K"], case["N"]
        share = torch.softmax(case["skew"] * torch.randn(G, generator=gen, device="cuda", dtype=torch.float64), 0)
        group = torch.multinomial(share, R, replacement=True, generator=gen)
        rows = torch.bincount(group, minlength=G)
        s["offsets"] = torch.cat([rows.new_zeros(1), rows.cumsum(0)]).to(torch.int32)
        s["longest"] = int(rows.max())  # the capacity that a program pads to
        s["A"] = _normal(gen, (R, K), dtype)
        s["W"] = _normal(gen, (G, K, N), dtype, K ** -0.5)
        if case["do"] == "train":
            s["grad"] = _normal(gen, (R, N), dtype)
            s["A"].requires_grad_(True)
            s["W"].requires_grad_(True)
    else:
        R, C = case["R"], case["C"]
        s["residual"] = _normal(gen, (R, C), dtype, 2.0)
        s["branch"] = _normal(gen, (R, C), dtype)
        s["gate"] = None if case["gate"] == "none" else _normal(gen, (R, C if case["gate"] == "full" else 1), dtype)
        s["scale"] = (0.3 + 0.1 * torch.randn(C, generator=gen, device="cuda")).to(dtype)
        s["weight_branch"] = (1.0 + 0.1 * torch.randn(C, generator=gen, device="cuda")).to(dtype)
        s["weight_output"] = (1.0 + 0.1 * torch.randn(C, generator=gen, device="cuda")).to(dtype)
        s["epsilon"] = 1e-5
        if case["do"] == "train":
            s["grad_stream"] = _normal(gen, (R, C), dtype)
            s["grad_normed"] = _normal(gen, (R, C), dtype)
            s["leaves"] = [t for t in _norm_arguments(s) if t is not None]
            s["leaves"] = [t.requires_grad_(True) for t in s["leaves"]]
    return s


def _norm_arguments(s):
    return s["residual"], s["branch"], s["gate"], s["scale"], s["weight_branch"], s["weight_output"]


# ------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return {"embedding": _own_embedding, "grouped": _own_grouped, "norm": _own_norm}[state["op"]](state)
    with torch.no_grad():
        return {"embedding": _plain_embedding, "grouped": _plain_grouped, "norm": _plain_norm}[state["op"]](state)


def _own_embedding(s):
    import mops_b200.torch as mt
    output = mt.embedding_lookup(s["W"], s["indices"], s["scale"])
    if s["do"] == "fwd":
        return output
    return output.detach(), *torch.autograd.grad(output, [s["W"]], s["grad"])


def _own_grouped(s):
    import mops_b200.torch as mt
    output = mt.grouped_matrix_product(s["A"], s["W"], s["offsets"])
    if s["do"] == "fwd":
        return output
    return output.detach(), *torch.autograd.grad(output, [s["A"], s["W"]], s["grad"])


def _own_norm(s):
    import mops_b200.torch as mt
    stream, normed = mt.gated_residual_norm(*_norm_arguments(s), s["epsilon"])
    if s["do"] == "fwd":
        return stream, normed
    return stream.detach(), normed.detach(), *torch.autograd.grad(
        [stream, normed], s["leaves"], [s["grad_stream"], s["grad_normed"]])


def _plain_embedding(s):
    W, indices = s["W"], s["indices"]
    output = (W[indices].float() * s["scale"]).to(W.dtype)
    if s["do"] == "fwd":
        return output
    sums = torch.zeros(W.shape, dtype=torch.float32, device=W.device)
    sums.index_add_(0, indices, s["grad"].float())
    return output, (sums * s["scale"]).to(W.dtype)


def _plain_grouped(s):
    # every group padded to the longest one, then a batched product
    A, W, offsets = s["A"], s["W"], s["offsets"].long()
    row = torch.arange(A.shape[0], device=A.device)
    group = torch.searchsorted(offsets, row, right=True) - 1
    within = row - offsets[group]
    at = offsets[:-1, None] + torch.arange(s["longest"], device=A.device)
    inside = (at < offsets[1:, None])[..., None]
    at = at.clamp(max=A.shape[0] - 1)
    padded, W32 = torch.where(inside, A[at].float(), 0.0), W.float()
    output = torch.bmm(padded, W32)[group, within].to(A.dtype)
    if s["do"] == "fwd":
        return output
    grad = torch.where(inside, s["grad"][at].float(), 0.0)
    grad_A = torch.bmm(grad, W32.transpose(1, 2))[group, within].to(A.dtype)
    return output, grad_A, torch.bmm(padded.transpose(1, 2), grad).to(W.dtype)


def _plain_norm(s):
    dtype = s["residual"].dtype
    x, b, g, scale, w, p = (None if t is None else t.float() for t in _norm_arguments(s))
    z = torch.sigmoid(g) if g is not None else torch.ones_like(x[:, :1])
    q = torch.rsqrt((b * b).mean(1, keepdim=True) + s["epsilon"])
    n = b * q
    y = x + scale * w * z * n
    r = torch.rsqrt((y * y).mean(1, keepdim=True) + s["epsilon"])
    outputs = [y, p * y * r]
    if s["do"] == "train":
        gh = s["grad_normed"].float()
        dh = p * gh
        dy = s["grad_stream"].float() + r * dh - y * r ** 3 * (dh * y).mean(1, keepdim=True)
        dn = dy * scale * w * z
        outputs += [dy, q * (dn - n * (dn * n).mean(1, keepdim=True))]
        if g is not None:
            dg = dy * scale * w * n * z * (1 - z)
            outputs.append(dg if g.shape[1] == x.shape[1] else dg.sum(1, keepdim=True))
        P = (dy * z * n).sum(0)
        outputs += [w * P, scale * P, (gh * y * r).sum(0)]
    return tuple(t.to(dtype) for t in outputs)


# ------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embedding": _exact_embedding, "grouped": _exact_grouped, "norm": _exact_norm}[case["op"]](s)


def _exact_embedding(s):
    W, indices = s["W"].double(), s["indices"].long()
    output = torch.index_select(W, 0, indices).mul_(s["scale"])
    if s["do"] == "fwd":
        return output
    # sums over the runs of equal tokens, as differences of the running sums at their ends
    order = torch.argsort(indices, stable=True)
    last = torch.bincount(indices, minlength=W.shape[0]).cumsum(0)
    gradient = torch.empty_like(W)
    for c in range(0, W.shape[1], 256):
        running = torch.zeros((indices.numel() + 1, min(256, W.shape[1] - c)), dtype=W.dtype, device=W.device)
        torch.cumsum(s["grad"][order, c:c + 256].double(), 0, out=running[1:])
        ends = running[last]
        gradient[:, c:c + 256] = torch.diff(ends, dim=0, prepend=torch.zeros_like(ends[:1])) * s["scale"]
    return output, gradient


def _exact_grouped(s):
    A, W = s["A"].double(), s["W"].double()
    bounds = s["offsets"].tolist()
    output = A.new_zeros((A.shape[0], W.shape[2]))
    gradients = [torch.zeros_like(A), torch.zeros_like(W)]
    for g, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        output[lo:hi] = A[lo:hi] @ W[g]
        if s["do"] == "train" and hi > lo:
            d = s["grad"][lo:hi].double()
            gradients[0][lo:hi] = d @ W[g].T
            gradients[1][g] = A[lo:hi].T @ d
    return output if s["do"] == "fwd" else (output, *gradients)


def _exact_norm(s):
    # the gradients by differentiating the definition, not by formulas
    leaves = [None if t is None else t.detach().double().requires_grad_(True) for t in _norm_arguments(s)]
    x, b, g, scale, w, p = leaves
    with torch.enable_grad():
        branch = b / (b.pow(2).mean(1, keepdim=True) + s["epsilon"]).sqrt() * w * scale
        y = x + (branch if g is None else branch / (1 + (-g).exp()))
        h = y / (y.pow(2).mean(1, keepdim=True) + s["epsilon"]).sqrt() * p
        if s["do"] == "fwd":
            return y.detach(), h.detach()
        gradients = torch.autograd.grad([y, h], [t for t in leaves if t is not None],
                                        [s["grad_stream"].double(), s["grad_normed"].double()])
    return y.detach(), h.detach(), *gradients


# ------------------------------------------------------------------------- what it costs
def work(case):
    """Bytes: every input read once (of a table, the rows that are asked for; of the matrices, those
    of groups that have rows) and every output written once."""
    size, train = BYTES[case["dtype"]], case["do"] == "train"
    if case["op"] == "embedding":
        T, V, D = case["T"], case["V"], case["D"]
        move = 4 * T + size * D * (min(T, V) + T)
        return {"bytes": move + (size * D * (T + V) if train else 0), "flops": T * D * (2 if train else 1)}
    if case["op"] == "grouped":
        R, G, K, N = case["R"], case["G"], case["K"], case["N"]
        move = size * (R * K + min(G, R) * K * N + R * N) + 4 * (G + 1)
        more = size * (R * N + R * K + G * K * N) if train else 0
        return {"bytes": move + more, "flops": 2 * R * K * N * (3 if train else 1)}
    R, C = case["R"], case["C"]
    gate = {"full": C, "row": 1, "none": 0}[case["gate"]]
    move = size * (R * (4 * C + gate) + 3 * C)
    more = size * (R * (4 * C + gate) + 3 * C) if train else 0
    return {"bytes": move + more, "flops": R * C * (40 if train else 14)}
