"""The operators of k2_amd/token_loss.py from their definitions in 64 bits, and how far a kernel that computes in 32 bits
may be from them.  Used by tests/test_token_loss_gpu.py and, on the host build of the kernels,
tests/test_cpu_build_token_loss.py.

Error budget, in units of U = 2^-24 (half a step of float32 at 1), for log p_i = ln2 (d_i - log2 s), d_i = (x_i - m) c:
  d_i: one rounding of the difference, one of c, one of the product: 3 |d_i|
  2^d_i: 3 |z_i| from its argument (z_i = ln2 d_i) and 4 of its own
  s: the terms weighted by p_i (sum p_i |z_i| <= log C) and one rounding for each addition; a lane adds at most 128 terms of
     its own, the tree and the join of the parts another 32: ADDS = 160
  so s is off by at most S = 3 sum p |z| + 4 + ADDS, log p_i by S + 8 |log p_i| + 4 and p_i by S + 3 |z_i| + 8 (times p_i).
A result in a narrower type is half a step of that type off besides, eps / 2 relative, or half its smallest value."""
import torch

U = 2.0 ** -24
ADDS = 160
NEG = float("-inf")
FLUSHED = 2.0 ** -125  # float32 exponentials below the smallest normal number may come out as 0


def logits_case(seed, rows, C, dtype, device, scale=2.0, peaks=4):
    """Rows as a trained model gives them: noise and a few likely tokens."""
    gen = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, C, generator=gen, device=device) * scale
    at = torch.randint(0, C, (rows, min(peaks, C)), generator=gen, device=device)
    x.scatter_(1, at, torch.rand(at.shape, generator=gen, device=device) * 9 + 1)
    return x.to(dtype)


class Softmax:
    """p, log p and the budgets above of rows x [rows, C] at a temperature."""

    def __init__(self, x, temperature=1.0):
        z = x.double() / temperature
        self.m = z.amax(1, keepdim=True)
        self.m = torch.where(self.m == NEG, torch.zeros_like(self.m), self.m)
        self.z = z - self.m
        e = self.z.exp()
        self.s = e.sum(1, keepdim=True)
        empty = self.s == 0  # a row that a mask left nothing of
        self.p = torch.where(empty, torch.zeros_like(e), e / self.s)
        self.logp = torch.where(empty, torch.full_like(e, NEG), self.z - self.s.log())
        z0 = torch.where(self.p > 0, self.z, torch.zeros_like(self.z))
        lp0 = torch.where(self.p > 0, self.logp, torch.zeros_like(self.z))
        self.entropy = -(self.p * lp0).sum(1, keepdim=True)
        spread = (self.p * z0.abs()).sum(1, keepdim=True)
        self.s_err = U * (3 * spread + 4 + ADDS)
        self.entropy_err = U * (3 * (self.p * z0 * z0).sum(1, keepdim=True) + (ADDS + 20) * spread + 8 * self.entropy) \
            + 2 * self.s_err
        self.p_rel = self.s_err + U * (3 * z0.abs() + 8)
        self.lp0 = lp0

    def logp_err(self, lp):
        return torch.where(torch.isfinite(lp), self.s_err + U * (8 * lp.abs() + 4), torch.zeros_like(lp))


def top(x, k):
    """Indices of the k largest, the lower index first where values are equal; past the C-th: -1."""
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :k]
    if order.shape[1] < k:
        order = torch.cat([order, torch.full((x.shape[0], k - order.shape[1]), -1, device=x.device)], 1)
    return order


def close(name, got, want, err):
    """|got - want| <= err, element by element; infinities and NaN have to be where they are wanted."""
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= err)
    assert not bad.any(), (name, int(bad.sum()), got[bad][:5], want[bad][:5], err.expand_as(want)[bad][:5])


def _narrow(dtype, want):
    """What rounding a result to dtype may add (subnormal results: half of the smallest value; float32 flushes them)."""
    info = torch.finfo(dtype)
    smallest = info.smallest_normal if dtype in (torch.float32, torch.bfloat16) else info.smallest_normal * info.eps
    return info.eps / 2 * want.abs() * (1 + 1e-6) + smallest


def check_token_logprobs(x, tokens, mask, temperature, k, got):
    """got: TokenLogprobs of rows x [rows, C]; tokens [rows, n] or None."""
    live = torch.ones(x.shape[0], 1, dtype=torch.bool, device=x.device) if mask is None else mask.reshape(-1, 1)
    x = torch.where(live, x.float(), torch.zeros((), device=x.device))
    sm = Softmax(x, temperature)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    if tokens is not None:
        there = (tokens >= 0) & live
        want = torch.where(there, sm.logp.gather(1, tokens.clamp(min=0)), zero)
        close("logprobs", got.logprobs.reshape(want.shape), want, sm.logp_err(want))
    if got.entropy is not None:
        want = torch.where(live, sm.entropy, zero)
        close("entropy", got.entropy.reshape(want.shape), want, sm.entropy_err)
    if k:
        order = torch.where(live, top(x, k), torch.full((), -1, device=x.device))
        assert torch.equal(got.top_tokens.reshape(order.shape), order), "top_tokens"
        want = torch.where(order >= 0, sm.logp.gather(1, order.clamp(min=0)), torch.full((), NEG, dtype=torch.float64, device=x.device))
        close("top_logprobs", got.top_logprobs.reshape(want.shape), want, sm.logp_err(want))


def check_token_grad(x, tokens, mask, temperature, grads, top_tokens, got):
    """grads: what reached logprobs [rows, n], entropy [rows, 1] and top_logprobs [rows, k], or None each."""
    live = torch.ones(x.shape[0], 1, dtype=torch.bool, device=x.device) if mask is None else mask.reshape(-1, 1)
    sm = Softmax(torch.where(live, x.float(), torch.zeros((), device=x.device)), temperature)
    lp_grad, h_grad, top_grad = [None if g is None else g.double() for g in grads]
    want, err = torch.zeros_like(sm.p), torch.zeros_like(sm.p)
    size = torch.zeros_like(sm.s)
    for entry, g in ((tokens, lp_grad), (top_tokens, top_grad)):
        if g is None:
            continue
        g = torch.where(entry >= 0, g, torch.zeros_like(g))
        want = (want - sm.p * g.sum(1, keepdim=True)).scatter_add(1, entry.clamp(min=0), g)
        size = size + g.abs().sum(1, keepdim=True)
        err = err.scatter_add(1, entry.clamp(min=0), 8 * U * g.abs())
    err = err + sm.p * size * (sm.p_rel + 140 * U)  # (the sum of up to 128 entries' gradients)
    if h_grad is not None:
        want = want - h_grad * sm.p * (sm.lp0 + sm.entropy)
        err = err + h_grad.abs() * sm.p * ((sm.lp0.abs() + sm.entropy) * (sm.p_rel + 8 * U) + sm.logp_err(sm.lp0) + sm.entropy_err)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    want = torch.where(live, want / temperature, zero)
    err = err / temperature + 4 * U * want.abs() + FLUSHED * (size + (0 if h_grad is None else 200 * h_grad.abs())) / temperature
    close("grad", got.reshape(want.shape), want, err + _narrow(got.dtype, want))


def distillation(x, top_logprobs, top_tokens, mask, temperature, bucket):
    """(row losses, their budget, gradient of each row's loss, its budget), of rows x [rows, C], lists [rows, K]."""
    rows, C = x.shape
    K = top_tokens.shape[1]
    live = torch.ones(rows, 1, dtype=torch.bool, device=x.device) if mask is None else mask.reshape(-1, 1)
    sm = Softmax(torch.where(live, x.float(), torch.zeros((), device=x.device)), temperature)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    there = (top_tokens >= 0) & live
    index = top_tokens.clamp(min=0)
    a = torch.where(there, top_logprobs.double(), torch.full((), NEG, dtype=torch.float64, device=x.device))
    a_err = 4 * U * torch.where(a > NEG, a.abs(), zero)
    some = there.any(1, keepdim=True)
    if not bucket:
        some = some & (a.amax(1, keepdim=True) > NEG)
        lse = torch.logsumexp(torch.where(some, a, zero), 1, keepdim=True)
        a = torch.where(some, a - lse, a)
        a_err = a_err + U * (4 * lse.abs() + K + 16)
    q = a.exp()
    q_err = q * (a_err + 4 * U)
    logp = sm.logp.gather(1, index)
    term = torch.where(q > 0, q * (a - logp), zero)
    loss = term.sum(1, keepdim=True)
    lp_err = sm.logp_err(logp)
    finite = torch.where(torch.isfinite(logp), logp, zero)
    a0 = torch.where(a > NEG, a, zero)
    loss_err = (q * (a_err + lp_err + 4 * U) + q_err * (a0 - finite).abs()).sum(1, keepdim=True) \
        + (K + 12) * U * torch.where(q > 0, q * (a0 - finite).abs(), zero).sum(1, keepdim=True)
    target = torch.zeros(rows, C, dtype=torch.float64, device=x.device)
    target_err = torch.zeros_like(target)
    column = torch.where(there, index, torch.zeros_like(index))
    target.scatter_add_(1, column, torch.where(there, q, zero))
    target_err.scatter_add_(1, column, torch.where(there, q_err + K * U * q, zero))
    mass = q.sum(1, keepdim=True)
    if bucket:
        listed = torch.zeros(rows, C, dtype=torch.float64, device=x.device).scatter_add_(1, column, there.double()) > 0
        rest_z = torch.where(listed, torch.full_like(sm.z, NEG), sm.z)
        high = rest_z.amax(1, keepdim=True)
        has = some & (high > NEG)
        high = torch.where(has, high, zero)
        rest_e = (rest_z - high).exp()
        rest_s = rest_e.sum(1, keepdim=True)
        log_p0 = torch.where(has, high + rest_s.log() - sm.s.log(), zero)
        q0 = torch.where(has, (1 - mass).clamp(min=0), zero)
        q0_err = U * (K + 12) + q_err.sum(1, keepdim=True)
        log_ratio = torch.where(q0 > 0, q0.log() - log_p0, zero)
        loss = loss + q0 * log_ratio
        away = torch.where(rest_e > 0, high - rest_z, zero)
        rest_err = U * (3 * (rest_e * away).sum(1, keepdim=True) / rest_s.clamp(min=1e-300) + 4 + ADDS)
        p0_rel = sm.s_err + rest_err + U * (8 * log_p0.abs() + 3 * high.abs() + 16)
        # d (q0 log q0) / d q0 = 1 + log q0: where q0 is as small as its error, the term moves by q0_err |log q0_err| < 18 q0_err
        loss_err = loss_err + torch.where(has, q0_err * (log_ratio.abs() + log_p0.abs() + 20) + q0 * (p0_rel + 8 * U), zero)
        share = torch.where(has, rest_e / rest_s.clamp(min=1e-300), zero)
        mass = mass + q0
        share_rel = rest_err + U * (3 * away + 12)
        grad = torch.where(listed, mass * sm.p - target, (mass * log_p0.exp() - q0) * share)
        p0 = torch.where(has, log_p0.exp(), zero)
        err = torch.where(listed, mass * sm.p * (sm.p_rel + (K + 20) * U) + target_err + sm.p * q0_err,
                          share * (q0_err * 2 + p0 * (p0_rel + 8 * U) + (mass * p0 - q0).abs() * share_rel))
    else:
        grad = sm.p - target
        err = sm.p * (sm.p_rel + 8 * U) + target_err
    grad = torch.where(some, grad, zero) / temperature
    err = torch.where(some, err, zero) / temperature + 6 * U * grad.abs() + FLUSHED * 4
    return (torch.where(some, loss, zero).squeeze(1), torch.where(some, loss_err, zero).squeeze(1), grad, err)


def check_distillation(x, top_logprobs, top_tokens, mask, temperature, bucket, got_loss, up, got_grad):
    """got_loss: the losses of the rows [rows]; got_grad: their gradient for ``up`` [rows] reaching them (or None)."""
    loss, loss_err, grad, err = distillation(x, top_logprobs, top_tokens, mask, temperature, bucket)
    close("loss", got_loss.reshape(-1), loss, loss_err)
    if got_grad is not None:
        up = up.double().reshape(-1, 1)
        want = grad * up
        close("grad", got_grad.reshape(want.shape), want, err * up.abs() + _narrow(got_grad.dtype, want))


def teacher_case(seed, x, K, temperature, holes=False, repeat=False, kept=None):
    """A list of K tokens a row with log-probs near the student's own: (top_logprobs, top_tokens)."""
    gen = torch.Generator(device=x.device).manual_seed(seed)
    rows, C = x.shape
    noisy = x.float() + torch.randn(rows, C, generator=gen, device=x.device)
    noisy = torch.where(noisy.isnan(), torch.zeros_like(noisy), noisy)
    lp = torch.log_softmax(noisy / temperature, 1)
    a, tokens = lp.topk(min(K, C), 1)
    if kept is not None:  # a given mass on the list
        a = a - torch.logsumexp(a, 1, keepdim=True) + torch.log(torch.full((), kept, device=x.device))
    if tokens.shape[1] < K:
        more = K - tokens.shape[1]
        tokens = torch.cat([tokens, tokens.new_full((rows, more), -1)], 1)
        a = torch.cat([a, a.new_full((rows, more), NEG)], 1)
    if repeat and K > 2:
        tokens[::3, 2] = tokens[::3, 0]
    if holes:
        gone = torch.rand(rows, K, generator=gen, device=x.device) < 0.3
        gone[:: 5] = True
        tokens = torch.where(gone, torch.full_like(tokens, -1), tokens)
        a = torch.where(gone, torch.full_like(a, NEG), a)
    return a.contiguous(), tokens.contiguous()
