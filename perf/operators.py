"""Cases and plain forms of the operators on a model's output logits: log-probs of given tokens with entropy and the
most likely alternatives (k2_amd.get_token_logprobs), and distillation from a teacher's listed log-probs
(k2_amd.distillation_loss, and k2_amd.rnnt_distillation_loss_pruned on the pruned lattice), each way.

``run`` computes a case in elementary torch operations in 32 bits, or, where ``own`` is true, with the calls a user
makes of the framework.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _case(name, kind, dtype, C, rows=0, B=0, T=0, R=0, tokens=0, top=0, entropy=False, K=0, rest="renormalise",
          reduction="mean", temperature=1.0, masked=False, holes=False):
    """kind: "score" (log-probs, nothing flows back), "train" (log-probs and the gradient), "distill" (loss and
    gradient), "lattice" (the same on the pruned lattice).  rows, or B x T x R rows of a pruned lattice; masked: part
    of the rows is padding (and holds NaN); holes: teacher lists with absent and repeated entries."""
    c = dict(kind=kind, dtype=dtype, C=C, rows=rows, B=B, T=T, R=R, tokens=tokens, top=top, entropy=entropy, K=K,
             rest=rest, reduction=reduction, temperature=temperature, masked=masked, holes=holes)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one step of a transducer's beam search: four hypotheses' joiner outputs, the best continuations of each
        _case("beam step", "score", "float32", 500, rows=4, tokens=0, top=4),
        # serving a language model: one sequence's next token out of a large vocabulary, with confidence
        _case("one token", "score", "bfloat16", 131072, rows=1, tokens=1, top=20, entropy=True),
        # a teacher labels the pruned lattice of the benchmark's pruned-loss shape, at a distillation temperature
        _case("label lattice", "score", "float32", 500, B=32, T=500, R=5, tokens=1, top=8, temperature=2.0, masked=True),
        # a teacher language model labels a batch of text with long lists
        _case("label text", "score", "bfloat16", 32000, rows=4096, tokens=1, top=64, entropy=True),
        # training a language model: cross entropy of the next token with an entropy term, padded batch, odd row count
        _case("train text", "train", "bfloat16", 32000, rows=8191, tokens=1, entropy=True, masked=True),
        # candidates of a rescoring pass trained against each other, rows of odd length that start anywhere
        _case("train odd", "train", "float16", 4999, rows=1013, tokens=3, top=5, entropy=True, temperature=0.7),
        # distillation of a small stateless predictor: a few rows, where the launches count
        _case("distill few", "distill", "float32", 500, rows=37, K=4),
        # distillation on the benchmark's pruned lattice, in both types that a joiner's logits come in
        _case("distill lattice", "lattice", "float32", 500, B=32, T=500, R=5, K=8, rest="bucket", reduction="sum", temperature=2.0),
        _case("distill lattice 16", "lattice", "bfloat16", 500, B=32, T=500, R=5, K=8, rest="bucket", reduction="mean"),
        # distillation of a language model from the twenty best tokens
        _case("distill text", "distill", "bfloat16", 32000, rows=8192, K=20),
        # the same out of a large vocabulary, with the rest of the mass in a bucket and a loss per row
        _case("distill large", "distill", "bfloat16", 131072, rows=2048, K=64, rest="bucket", reduction="none"),
        # lists with absent and repeated entries, odd row length, padding
        _case("distill odd", "distill", "float16", 1237, rows=3001, K=17, rest="bucket", reduction="none",
              temperature=3.0, masked=True, holes=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "train", "distill", "lattice"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    most = 1 << 27  # logits of a case
    C = _log_uniform(rng, 40, 131072 if kind != "lattice" else 5000)
    tau = rng.choice([1.0, 1.0, 0.5, 2.0, 3.3])
    if kind == "lattice":
        B, R = rng.randint(1, 32), rng.randint(2, 6)
        T = _log_uniform(rng, 8, max(9, min(700, most // (B * R * C))))
        return _case(None, kind, dtype, C, B=B, T=T, R=R, K=rng.randint(1, 24), rest=rng.choice(["renormalise", "bucket"]),
                     reduction=rng.choice(["none", "sum", "mean"]), temperature=tau, holes=rng.random() < 0.3)
    rows = _log_uniform(rng, 1, max(2, min(100000, most // C)))
    masked = rng.random() < 0.4 and rows > 4
    if kind == "distill":
        K = _log_uniform(rng, 1, min(128, C // 4))
        return _case(None, kind, dtype, C, rows=rows, K=K, rest=rng.choice(["renormalise", "bucket"]),
                     reduction=rng.choice(["none", "sum", "mean"]), temperature=tau, masked=masked, holes=rng.random() < 0.3)
    tokens = rng.choice([1, 1, 1, 2, 5])
    top = rng.choice([0, 0, 1, 4, 10, 20, 33, 64]) if kind == "score" else rng.choice([0, 0, 0, 3])
    return _case(None, kind, dtype, C, rows=rows, tokens=tokens, top=min(top, C), entropy=rng.random() < 0.6,
                 temperature=tau, masked=masked)


def _rows(case):
    return case["rows"] or case["B"] * case["T"] * case["R"]


def _lengths(case):
    """Frames of each sequence of a padded batch of lattices: from all of T down to three fifths of it."""
    B, T = case["B"], case["T"]
    return [T - (b * (2 * T // 5)) // max(B - 1, 1) for b in range(B)]


def _live_rows(case):
    """How many rows are not padding: the same for every seed."""
    if case["kind"] == "lattice" or (case["B"] and case["masked"]):
        return sum(_lengths(case)) * case["R"]
    return _rows(case) - _rows(case) // 5 if case["masked"] else _rows(case)


def work(case):
    rows, live, C = _rows(case), _live_rows(case), case["C"]
    size = 4 if case["dtype"] == "float32" else 2
    moved = live * C * size
    if case["kind"] in ("score", "train"):
        moved += live * (case["tokens"] * 12 + case["top"] * 12 + (4 if case["entropy"] else 0))
        ops = (7.0 if case["entropy"] else 5.0) * live * C
        if case["kind"] == "train":
            moved += rows * C * size + live * (4 * case["tokens"] + 4 * case["top"] + (4 if case["entropy"] else 0))
            ops *= 2
    else:
        moved += live * (case["K"] * 12 + 4) + rows * C * size
        ops = 10.0 * live * C
    return {"bytes": float(moved), "flops": float(ops)}


# ---- inputs -------------------------------------------------------------------------------------


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rows, C, dtype = _rows(case), case["C"], DTYPES[case["dtype"]]
    rand = lambda *shape: torch.rand(*shape, generator=gen, device=dev)  # noqa: E731
    logits = torch.randn(rows, C, generator=gen, device=dev).mul_(1.5)
    state = {"case": case, "mask": None}
    # a handful of likely tokens in each row, as trained models give them
    likely = max(case["K"], min(8, C // 4))
    at = (torch.randint(0, C, (rows, 1), generator=gen, device=dev)
          + torch.arange(likely, device=dev) * (C // likely)) % C
    height = rand(rows, likely).mul_(7.0).sort(dim=1, descending=True).values
    logits.scatter_add_(1, at, height + 2.0)
    if case["kind"] in ("score", "train"):
        n = case["tokens"]
        which = torch.randint(0, likely, (rows, max(n, 1)), generator=gen, device=dev)
        tokens = at.gather(1, which)
        state["tokens"] = None if n == 0 else tokens[:, 0].contiguous() if n == 1 else tokens
        state["lp_grad"] = torch.randn(*((rows,) if n == 1 else (rows, n)), generator=gen, device=dev)
        state["entropy_grad"] = torch.randn(rows, generator=gen, device=dev) * 0.1
        state["top_grad"] = torch.randn(rows, case["top"], generator=gen, device=dev) * 0.3
    else:
        K = case["K"]
        tokens = at[:, :K].contiguous()
        scores = height[:, :K] / case["temperature"] + torch.randn(rows, K, generator=gen, device=dev) * 0.5
        kept = 1.0 - torch.pow(10.0, -0.3 - 3.5 * rand(rows, 1))  # the mass on the list
        logprobs = scores - torch.logsumexp(scores, 1, keepdim=True) + kept.log()
        if case["holes"]:
            absent = rand(rows, K) < 0.2
            absent |= rand(rows, 1) < 0.05  # rows without any entry
            tokens = torch.where(absent, torch.full_like(tokens, -1), tokens)
            logprobs = torch.where(absent, torch.full_like(logprobs, float("-inf")), logprobs)
            if K > 2:
                again = rand(rows) < 0.1
                tokens[:, 1] = torch.where(again & (tokens[:, 0] >= 0) & (tokens[:, 1] >= 0), tokens[:, 0], tokens[:, 1])
        state["top_tokens"], state["top_logprobs"] = tokens, logprobs
        groups = case["B"] if case["kind"] == "lattice" else rows
        state["loss_grad"] = (torch.randn(groups, generator=gen, device=dev) if case["reduction"] == "none"
                              else torch.full((), 0.25, device=dev))
    dead = None
    if case["B"]:
        B, T, R = case["B"], case["T"], case["R"]
        S = max(R, T // 5)
        frames = torch.tensor(_lengths(case), device=dev)
        # where each frame's window starts: from row 0 to the last ones of the sequence, evenly
        start = (torch.arange(T, device=dev).unsqueeze(0) * (S + 1 - R) // frames.unsqueeze(1)).clamp(max=S + 1 - R)
        state["ranges"] = (start.unsqueeze(2) + torch.arange(R, device=dev)).contiguous()
        boundary = torch.zeros(B, 4, dtype=torch.int64, device=dev)
        boundary[:, 2], boundary[:, 3] = S, frames
        state["boundary"] = boundary
        live = (torch.arange(T, device=dev).unsqueeze(0) < frames.unsqueeze(1)).unsqueeze(2).expand(B, T, R).contiguous()
        if case["masked"]:
            state["mask"] = live
        if case["masked"] or case["kind"] == "lattice":
            dead = ~live.reshape(rows)
    elif case["masked"]:
        order = torch.randperm(rows, generator=gen, device=dev)
        live = torch.ones(rows, dtype=torch.bool, device=dev)
        live[order[: rows // 5]] = False
        state["mask"], dead = live, ~live
    if dead is not None:  # what a padded batch holds behind its sequences is anything
        logits.masked_fill_(dead.unsqueeze(1), float("nan"))
    logits = logits.to(dtype)
    if case["B"]:
        lead = (case["B"], case["T"], case["R"])
        for name in ("tokens", "lp_grad", "entropy_grad", "top_grad", "top_tokens", "top_logprobs"):
            if state.get(name) is not None:
                state[name] = state[name].reshape(lead + state[name].shape[1:])
        logits = logits.reshape(lead + (C,))
    state["logits"] = logits
    return state


# ---- the operators ------------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if case["kind"] == "score":
        return _own_score(state) if own else _plain_score(state)
    if case["kind"] == "train":
        return _own_train(state) if own else _plain_train(state)
    return _own_distill(state) if own else _plain_distill(state)


def _named(case, logprobs, entropy, top_logprobs, top_tokens):
    out = {}
    if case["tokens"]:
        out["logprobs"] = logprobs
    if case["entropy"]:
        out["entropy"] = entropy
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = top_logprobs, top_tokens
    return out


def _own_score(state):
    import k2_amd
    case = state["case"]
    return _named(case, *k2_amd.get_token_logprobs(state["logits"], state["tokens"], mask=state["mask"],
                                                   temperature=case["temperature"], num_top=case["top"],
                                                   return_entropy=case["entropy"]))


def _own_train(state):
    import k2_amd
    case = state["case"]
    logits = state["logits"].detach().requires_grad_(True)
    got = k2_amd.get_token_logprobs(logits, state["tokens"], mask=state["mask"], temperature=case["temperature"],
                                    num_top=case["top"], return_entropy=case["entropy"])
    outputs, grads = [got.logprobs], [state["lp_grad"]]
    if case["entropy"]:
        outputs.append(got.entropy)
        grads.append(state["entropy_grad"])
    if case["top"]:
        outputs.append(got.top_logprobs)
        grads.append(state["top_grad"])
    (grad,) = torch.autograd.grad(outputs, logits, grads)
    return dict(_named(case, *(None if t is None else t.detach() for t in got)), grad=grad)


def _own_distill(state):
    import k2_amd
    case = state["case"]
    logits = state["logits"].detach().requires_grad_(True)
    how = dict(temperature=case["temperature"], rest=case["rest"], reduction=case["reduction"])
    if case["kind"] == "lattice":
        loss = k2_amd.rnnt_distillation_loss_pruned(logits, state["top_logprobs"], state["top_tokens"], state["ranges"],
                                                    state["boundary"], **how)
    else:
        loss = k2_amd.distillation_loss(logits, state["top_logprobs"], state["top_tokens"], mask=state["mask"], **how)
    (grad,) = torch.autograd.grad(loss, logits, state["loss_grad"])
    return {"loss": loss.detach(), "grad": grad}


def _softmax(logits, live, temperature):
    """d = (x - max x) / temperature, e = exp(d), their sum, and log p: rows that are not live count as zeros."""
    x = logits.float()
    if live is not None:
        x = torch.where(live.unsqueeze(-1), x, torch.zeros((), device=x.device))
    d = (x - x.amax(-1, keepdim=True)) / temperature
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    return x, d, e, total, d - total.log()


def _best(x, k):
    """The k largest of each row, the lower index first where values are equal: the order of the values and the index
    in one whole number."""
    bits = (x + 0.0).view(torch.int32).to(torch.int64)
    order = torch.where(bits < 0, -2147483649 - bits, bits)
    key = order * 4294967296 + (4294967295 - torch.arange(x.shape[-1], device=x.device))
    return 4294967295 - (key.topk(k, dim=-1, sorted=True).values & 4294967295)


def _plain_score(state, pieces=None):
    case, live = state["case"], state["mask"]
    x, d, e, total, logp = pieces or _softmax(state["logits"], live, case["temperature"])
    logprobs = entropy = top_logprobs = top_tokens = None
    if case["tokens"]:
        tokens = state["tokens"]
        many = tokens.dim() == x.dim()
        logprobs = logp.gather(-1, tokens if many else tokens.unsqueeze(-1))
        if live is not None:
            logprobs = logprobs * live.unsqueeze(-1)
        logprobs = logprobs if many else logprobs.squeeze(-1)
    if case["entropy"]:
        entropy = (total.log() - (d * e).sum(-1, keepdim=True) / total).squeeze(-1)
        if live is not None:
            entropy = entropy * live
    if case["top"]:
        top_tokens = _best(x, case["top"])
        top_logprobs = logp.gather(-1, top_tokens)
        if live is not None:
            top_tokens = torch.where(live.unsqueeze(-1), top_tokens, torch.full_like(top_tokens, -1))
            top_logprobs = torch.where(live.unsqueeze(-1), top_logprobs, torch.full_like(top_logprobs, float("-inf")))
    return _named(case, logprobs, entropy, top_logprobs, top_tokens)


def _plain_train(state):
    case, live = state["case"], state["mask"]
    pieces = _softmax(state["logits"], live, case["temperature"])
    out = _plain_score(state, pieces)
    _, _, e, total, logp = pieces
    p = e / total
    rows = p.shape[:-1]
    entries, grads = [state["tokens"].reshape(rows + (-1,))], [state["lp_grad"].reshape(rows + (-1,))]
    if case["top"]:
        entries.append(out["top_tokens"].clamp(min=0))
        grads.append(state["top_grad"])
    entries, grads = torch.cat(entries, -1), torch.cat(grads, -1)
    grad = -p * grads.sum(-1, keepdim=True)
    if case["entropy"]:
        grad = grad - state["entropy_grad"].unsqueeze(-1) * p * (logp + out["entropy"].unsqueeze(-1))
    grad = grad.scatter_add(-1, entries, grads) / case["temperature"]
    if live is not None:
        grad = grad * live.unsqueeze(-1)
    out["grad"] = grad.to(state["logits"].dtype)
    return out


def _lattice_live(state):
    """Rows of the pruned lattice that lie in their sequence's box."""
    ranges, box = state["ranges"], state["boundary"][:, None, None, :]
    t = torch.arange(ranges.shape[1], device=ranges.device)[None, :, None]
    return (t >= box[..., 1]) & (t < box[..., 3]) & (ranges >= box[..., 0]) & (ranges <= box[..., 2])


def _plain_distill(state):
    case = state["case"]
    live = _lattice_live(state) if case["kind"] == "lattice" else state["mask"]
    tokens, a = state["top_tokens"], state["top_logprobs"]
    x, d, e, total, logp = _softmax(state["logits"], live, case["temperature"])
    present = tokens >= 0
    if live is not None:
        present = present & live.unsqueeze(-1)
    index = tokens.clamp(min=0)
    a = torch.where(present, a, torch.full_like(a, float("-inf")))
    zero = torch.zeros((), device=x.device)
    some = present.any(-1, keepdim=True)
    if case["rest"] == "renormalise":
        high = torch.where(some, a.amax(-1, keepdim=True), zero)
        mass = (a - high).exp().sum(-1, keepdim=True)
        a = torch.where(present, a - high - mass.log(), a)
    q = a.exp()
    rows = torch.where(q > 0, q * (a - logp.gather(-1, index)), zero).sum(-1)
    p = e / total
    # entries that are not there add nothing, wherever their index points
    listed_q = torch.zeros_like(x).scatter_add_(-1, index, q)
    if case["rest"] == "renormalise":
        grad = torch.where(some, p - listed_q, zero)
    else:
        q0 = (1.0 - q.double().sum(-1, keepdim=True)).clamp(min=0.0).float()  # a difference of nearly equal numbers
        q0 = torch.where(some, q0, zero)
        listed_any = torch.zeros_like(x).scatter_add_(-1, index, present.float()) > 0
        rest = torch.where(listed_any, torch.full_like(d, float("-inf")), d)
        high = rest.amax(-1, keepdim=True)
        rest_e = (rest - high).exp()
        rest_sum = rest_e.sum(-1, keepdim=True)
        log_p0 = high + rest_sum.log() - total.log()
        rows = rows + torch.where(q0 > 0, q0 * (q0.log() - log_p0), zero).squeeze(-1)
        mass = q.sum(-1, keepdim=True) + q0
        grad = torch.where(listed_any, mass * p - listed_q, (mass * log_p0.exp() - q0) * (rest_e / rest_sum))
        grad = torch.where(some, grad, zero)
    scale, reduction = state["loss_grad"], case["reduction"]
    if case["kind"] == "lattice":
        rows = rows.sum((1, 2))
        loss = rows if reduction == "none" else rows.sum() if reduction == "sum" else rows.mean()
        scale = scale.reshape(-1, 1, 1, 1) / (rows.shape[0] if reduction == "mean" else 1.0)
    else:
        count = (live.sum().clamp(min=1) if live is not None else rows.numel()) if reduction == "mean" else 1.0
        loss = rows if reduction == "none" else rows.sum() / count
        scale = scale.unsqueeze(-1) / count
    return {"loss": loss, "grad": (grad * (scale / case["temperature"])).to(state["logits"].dtype)}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    C = case["C"]
    x = state["logits"].reshape(-1, C)
    lead = tuple(state["logits"].shape[:-1])
    if case["kind"] == "lattice":
        inside = torch.zeros(lead, dtype=torch.bool, device=x.device)
        S = int(state["boundary"][0, 2])
        for b, frames in enumerate(_lengths(case)):
            inside[b, :frames] = state["ranges"][b, :frames] <= S
        live = inside.reshape(-1)
    else:
        live = (torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if state["mask"] is None
                else state["mask"].reshape(-1))
    if case["kind"] in ("score", "train"):
        return _exact_scores(case, state, x, live, lead)
    return _exact_distill(case, state, x, live, lead)


def _pieces(n, C):
    """Row ranges of about 2^26 logits."""
    step = max(1, (1 << 26) // C)
    return [(i, min(n, i + step)) for i in range(0, n, step)]


def _exact_scores(case, state, x, live, lead):
    n, k = case["tokens"], case["top"]
    tokens = state["tokens"].reshape(x.shape[0], -1) if n else None
    parts = {"logprobs": [], "entropy": [], "top_logprobs": [], "top_tokens": [], "grad": []}
    for lo, hi in _pieces(*x.shape):
        on = live[lo:hi].unsqueeze(1)
        lp = torch.log_softmax(x[lo:hi].double().masked_fill(~on, 0.0) / case["temperature"], dim=1)
        p = lp.exp()
        h = -(p * lp).sum(1, keepdim=True)
        g = torch.zeros_like(lp)
        if n:
            parts["logprobs"].append(lp.gather(1, tokens[lo:hi]).masked_fill(~on, 0.0))
            if case["kind"] == "train":
                up = state["lp_grad"].reshape(x.shape[0], -1)[lo:hi].double()
                for j in range(n):
                    g -= up[:, j:j + 1] * p
                    g.scatter_add_(1, tokens[lo:hi, j:j + 1], up[:, j:j + 1])
        if case["entropy"]:
            parts["entropy"].append(h.masked_fill(~on, 0.0))
            if case["kind"] == "train":
                g -= state["entropy_grad"].reshape(-1, 1)[lo:hi].double() * p * (lp + h)
        if k:
            order = torch.sort(x[lo:hi].float().masked_fill(~on, 0.0), dim=1, descending=True, stable=True).indices[:, :k]
            best = lp.gather(1, order)
            parts["top_logprobs"].append(best.masked_fill(~on, float("-inf")))
            parts["top_tokens"].append(order.masked_fill(~on, -1))
            if case["kind"] == "train":
                up = state["top_grad"].reshape(-1, k)[lo:hi].double()
                g -= up.sum(1, keepdim=True) * p
                g.scatter_add_(1, order, up)
        if case["kind"] == "train":
            parts["grad"].append((g / case["temperature"]).masked_fill(~on, 0.0))
    out = {}
    if n:
        out["logprobs"] = torch.cat(parts["logprobs"]).reshape(lead + (() if n == 1 else (n,)))
    if case["entropy"]:
        out["entropy"] = torch.cat(parts["entropy"]).reshape(lead)
    if k:
        out["top_logprobs"] = torch.cat(parts["top_logprobs"]).reshape(lead + (k,))
        out["top_tokens"] = torch.cat(parts["top_tokens"]).reshape(lead + (k,))
    if case["kind"] == "train":
        out["grad"] = torch.cat(parts["grad"]).reshape(lead + (case["C"],))
    return out


def _exact_distill(case, state, x, live, lead):
    tokens = state["top_tokens"].reshape(x.shape[0], -1)
    given = state["top_logprobs"].reshape(x.shape[0], -1).double()
    there = (tokens >= 0) & live.unsqueeze(1)
    some = there.any(1)
    a = given.masked_fill(~there, float("-inf"))
    if case["rest"] == "renormalise":
        a = torch.where(some.unsqueeze(1), torch.log_softmax(a.masked_fill(~some.unsqueeze(1), 0.0), dim=1), a)
    q = a.exp()
    bucket = (1.0 - q.sum(1)).clamp(min=0.0) * some if case["rest"] == "bucket" else torch.zeros_like(q[:, 0])
    losses, grads = [], []
    for lo, hi in _pieces(*x.shape):
        lp = torch.log_softmax(x[lo:hi].double().masked_fill(~live[lo:hi].unsqueeze(1), 0.0) / case["temperature"], dim=1)
        at, on, qq = tokens[lo:hi].clamp(min=0), there[lo:hi], q[lo:hi]
        # the target's probability of each token, and which tokens are on the list (column C takes what is not there)
        column = torch.where(on, at, torch.full_like(at, case["C"]))
        target = torch.zeros(hi - lo, case["C"] + 1, dtype=torch.float64, device=x.device).scatter_add_(1, column, qq)[:, :-1]
        is_listed = torch.zeros(hi - lo, case["C"] + 1, dtype=torch.bool, device=x.device).scatter_(1, column, True)[:, :-1]
        loss = torch.where(on & (qq > 0), qq * (a[lo:hi] - lp.gather(1, at)), 0.0).sum(1)
        q0 = bucket[lo:hi]
        if case["rest"] == "bucket":
            log_p0 = torch.logsumexp(lp.masked_fill(is_listed, float("-inf")), dim=1)
            loss = loss + torch.where(q0 > 0, q0 * (q0.log() - log_p0), 0.0)
            share = (lp - log_p0.unsqueeze(1)).exp().masked_fill(is_listed, 0.0)
            target = target + q0.unsqueeze(1) * share
        grad = (target.sum(1, keepdim=True) * lp.exp() - target) * some[lo:hi].unsqueeze(1)
        losses.append(loss)
        grads.append(grad)
    rows, grad = torch.cat(losses), torch.cat(grads)
    up, reduction = state["loss_grad"].double(), case["reduction"]
    if case["kind"] == "lattice":
        rows = rows.reshape(case["B"], -1).sum(1)
        if reduction != "none":
            rows = rows.sum() if reduction == "sum" else rows.sum() / case["B"]
            up = up / (case["B"] if reduction == "mean" else 1)
        up = up.expand(case["B"]).repeat_interleave(case["T"] * case["R"]).unsqueeze(1)
    else:
        if reduction != "none":
            n = max(int(live.sum()), 1) if reduction == "mean" else 1
            rows, up = rows.sum() / n, up / n
        up = up.unsqueeze(-1)
    grad = grad * up / case["temperature"]
    return {"loss": rows.reshape(lead) if reduction == "none" and case["kind"] != "lattice" else rows,
            "grad": grad.reshape(lead + (case["C"],))}
