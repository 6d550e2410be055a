"""k2_amd/token_loss.py on the GPU against its definitions in 64 bits (tests/token_oracle.py, where the tolerances are
derived): types, row lengths, strides, masks, lists, gradients, streams and graphs."""
import math

import pytest
import torch

import token_oracle as orc

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NEG = float("-inf")


def _mask(seed, rows, device):
    gen = torch.Generator(device=device).manual_seed(seed)
    return torch.rand(rows, generator=gen, device=device) < 0.7


def _scores(x, tokens, mask, temperature, k, entropy=True):
    import k2_amd as k2
    got = k2.get_token_logprobs(x, tokens, mask=mask, temperature=temperature, num_top=k, return_entropy=entropy)
    two_d = None if tokens is None else tokens.reshape(x.shape[0], -1)
    orc.check_token_logprobs(x, two_d, mask, temperature, k, got)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 2, 3, 5, 8, 9, 63, 64, 65, 500, 511, 1000, 1237, 2047, 2048, 2049, 4999, 8200, 16385, 32000,
                               50001, 65536, 131071, 131072, 200003])
def test_forward_over_row_lengths(device, dtype, C):
    rows = 7
    x = orc.logits_case(C, rows, C, dtype, device)
    tokens = torch.randint(0, C, (rows, 2), device=device)
    tokens[1, 0] = -1
    for k in (0, 1, 4, 20, 64):
        _scores(x, tokens, _mask(C, rows, device) if k == 4 else None, 1.0 if k < 20 else 0.6, k)


@pytest.mark.parametrize("rows", [1, 2, 5, 64, 1000, 5003])
@pytest.mark.parametrize("C", [30, 500, 3000])
def test_forward_over_row_counts(device, rows, C):
    x = orc.logits_case(rows, rows, C, torch.bfloat16, device)
    _scores(x, torch.randint(0, C, (rows,), device=device), _mask(rows, rows, device), 2.0, 8)
    _scores(x.float(), None, None, 1.0, 10, entropy=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [40, 700, 9000, 70000])
def test_ties_and_masked_vocabularies(device, dtype, C):
    """The order of equal logits, and rows that hold little: constant rows, a few distinct values, an allow-list of three
    tokens in front of -inf or of the type's lowest value, a contiguous range of tokens, nothing at all."""
    lowest = torch.finfo(dtype).min
    x = torch.zeros(12, C, dtype=dtype, device=device)
    gen = torch.Generator(device=device).manual_seed(C)
    x[1] = 3.25
    x[2] = torch.randint(0, 4, (C,), generator=gen, device=device).to(dtype)
    x[3] = torch.where(torch.rand(C, generator=gen, device=device) < 0.01, 1.0, 0.0).to(dtype)
    x[4] = NEG
    x[4, [C // 3, C // 2, C - 1]] = torch.tensor([1.0, -2.0, 1.0], dtype=dtype, device=device)
    x[5] = lowest
    x[5, [0, C // 2]] = torch.tensor([0.5, 0.25], dtype=dtype, device=device)
    x[6] = NEG
    x[6, C // 4: C // 2] = torch.randn(C // 2 - C // 4, generator=gen, device=device).to(dtype)
    x[7] = NEG
    x[8] = lowest
    x[9] = torch.arange(C, device=device).to(dtype) if dtype == torch.float32 else torch.arange(C, device=device).remainder(37).to(dtype)
    x[10] = -x[9]
    x[11, ::2] = -0.0  # equal to 0: the lower index first
    tokens = torch.tensor([0, C // 3, C - 1], device=device).repeat(12, 1)
    for k in (1, 7, 20, 64):
        _scores(x, tokens, None, 1.0, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [60, 700, 5000, 40001])
def test_far_from_zero(device, dtype, C):
    """Rows that lie anywhere in the type's range, and temperatures that take the logits far apart or close together: the
    budgets are those of differences of logits, wherever the logits are."""
    import k2_amd as k2
    x = orc.logits_case(C, 8, C, torch.float32, device)
    offsets = [0.0, 300.0, -3000.0, 4.0e4, -6.0e4] + ([2.0e6, -1.0e9, 3.0e20] if dtype != torch.float16 else [100.0, -100.0, 1.0e3])
    x = (x + torch.tensor(offsets, device=device).unsqueeze(1)).to(dtype).requires_grad_()
    tokens = torch.randint(0, C, (8, 1), device=device)
    for temperature in (1.0, 0.01, 1.0e-9, 1.0e6):
        got = k2.get_token_logprobs(x, tokens, temperature=temperature, num_top=4, return_entropy=True)
        orc.check_token_logprobs(x.detach(), tokens, None, temperature, 4, k2.TokenLogprobs(*(u.detach() for u in got)))
        up = torch.ones_like(got.logprobs)
        (grad,) = torch.autograd.grad(got.logprobs, x, up)
        if temperature >= 0.01:  # (beyond, the gradient itself leaves float16)
            orc.check_token_grad(x.detach(), tokens, None, temperature, (up, None, None), None, grad)
        without = k2.get_token_logprobs(x.detach(), tokens, temperature=temperature, return_entropy=True)
        orc.check_token_logprobs(x.detach(), tokens, None, temperature, 0, without)
    a, t = orc.teacher_case(1, x.detach(), 5, 1.0)
    for bucket in (False, True):
        loss = k2.distillation_loss(x, a, t, rest="bucket" if bucket else "renormalise", reduction="none")
        (grad,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
        orc.check_distillation(x.detach(), a, t, None, 1.0, bucket, loss.detach(), torch.ones_like(loss), grad)


def test_more_rows_than_a_launch_takes(device):
    """Calls beyond 2^20 rows are several launches; the gradient's go from the last rows to the first."""
    import k2_amd as k2
    rows, C = (1 << 20) + 1037, 9
    x = orc.logits_case(4, rows, C, torch.float16, device).requires_grad_()
    tokens = torch.randint(0, C, (rows, 1), device=device)
    mask = _mask(1, rows, device)
    got = k2.get_token_logprobs(x, tokens, mask=mask, num_top=2, return_entropy=True)
    orc.check_token_logprobs(x.detach(), tokens, mask, 1.0, 2, k2.TokenLogprobs(*(u.detach() for u in got)))
    up = torch.randn(rows, 1, device=device)
    (grad,) = torch.autograd.grad(got.logprobs, x, up)
    orc.check_token_grad(x.detach(), tokens, mask, 1.0, (up, None, None), None, grad)
    a, t = orc.teacher_case(2, x.detach(), 3, 1.0)
    loss = k2.distillation_loss(x, a, t, mask=mask, rest="bucket", reduction="none")
    up = torch.randn(rows, device=device)
    (grad,) = torch.autograd.grad(loss, x, up)
    orc.check_distillation(x.detach(), a, t, mask, 1.0, True, loss.detach(), up, grad)
    total = k2.distillation_loss(x, a, t, mask=mask, rest="bucket", reduction="sum")
    assert abs(total.double() - loss.double().sum()) <= 1e-6 * loss.double().abs().sum()


@pytest.mark.parametrize("dtype", DTYPES)
def test_not_numbers(device, dtype):
    """NaN and +inf make their row's results NaN and no other's; a NaN is listed before every number; rows masked out may
    hold anything."""
    import k2_amd as k2
    C = 300
    x = orc.logits_case(5, 6, C, dtype, device)
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    x[3] = float("nan")
    mask = torch.tensor([True, True, True, False, True, True], device=device)
    tokens = torch.zeros(6, dtype=torch.int64, device=device)
    got = k2.get_token_logprobs(x, tokens, mask=mask, num_top=5, return_entropy=True)
    for r in (1, 2):
        assert got.logprobs[r].isnan() and got.entropy[r].isnan() and got.top_logprobs[r].isnan().all()
    assert got.top_tokens[1, 0] == 7 and got.top_tokens[2, 0] == 9
    assert torch.equal(got.top_tokens[1:3], orc.top(torch.nan_to_num(x[1:3], nan=1e30, posinf=1e30), 5))
    keep = [0, 3, 4, 5]
    orc.check_token_logprobs(x[keep], tokens[keep].unsqueeze(1), mask[keep], 1.0, 5,
                             k2.TokenLogprobs(*(t[keep] for t in got)))


def test_tokens_outside_the_vocabulary(device):
    """Negative: absent, log-prob 0 and no gradient.  Past the end: NaN in its log-prob and its row's gradient."""
    import k2_amd as k2
    x = orc.logits_case(1, 4, 50, torch.float32, device).requires_grad_()
    tokens = torch.tensor([[3, -1], [-5, -1], [50, 2], [49, 1 << 40]], device=device)
    got = k2.get_token_logprobs(x, tokens).logprobs
    want = torch.log_softmax(x.detach().double(), 1)
    assert got[0, 1] == 0 and got[1].eq(0).all() and got[2, 0].isnan() and got[3, 1].isnan()
    torch.testing.assert_close(got[3, 0].double(), want[3, 49], rtol=1e-5, atol=1e-5)
    (grad,) = torch.autograd.grad(got[:2].sum(), x)
    assert grad[1].eq(0).all() and grad[2:].isnan().all()  # (a gradient of 0 for a wrong token is still NaN)
    lists = torch.full((4, 1), -0.5, device=device)
    loss = k2.distillation_loss(x, lists, tokens[:, :1], reduction="none")
    assert loss[2].isnan() and loss[1] == 0 and torch.isfinite(loss[[0, 1, 3]]).all()
    (grad,) = torch.autograd.grad(loss[[0, 1, 3]].sum(), x)
    assert grad[2].isnan().all() and torch.isfinite(grad[[0, 1, 3]]).all()


def _strided(x, how):
    """The values of x [rows, C] in a tensor of other strides."""
    rows, C = x.shape
    if how == "padded vocabulary":
        return torch.full((rows, C + 13), 7.0, dtype=x.dtype, device=x.device).index_copy_(
            1, torch.arange(C, device=x.device), x)[:, :C]
    if how == "odd start":
        buf = torch.full((rows * C + 3,), 7.0, dtype=x.dtype, device=x.device)
        buf[1:1 + rows * C] = x.reshape(-1)
        return buf[1:1 + rows * C].view(rows, C)
    if how == "last positions":
        buf = torch.full((rows, 3, C), 7.0, dtype=x.dtype, device=x.device)
        buf[:, -1] = x
        return buf[:, -1]
    assert how == "columns"
    return x.t().contiguous().t()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("how", ["padded vocabulary", "odd start", "last positions", "columns"])
@pytest.mark.parametrize("C", [37, 501, 2500, 33001])
def test_strides(device, dtype, how, C):
    import k2_amd as k2
    rows = 6
    x = orc.logits_case(C, rows, C, dtype, device)
    y = _strided(x, how)
    assert torch.equal(x, y)
    tokens = torch.randint(0, C, (rows,), device=device)
    a, t = orc.teacher_case(3, x, 5, 1.0)
    results = []
    for z in (x.clone().requires_grad_(), y.detach().requires_grad_()):
        got = k2.get_token_logprobs(z, tokens, num_top=4, return_entropy=True)
        (grad,) = torch.autograd.grad([got.logprobs.sum(), got.entropy.sum()], z)
        loss = k2.distillation_loss(z, a, t, rest="bucket", reduction="none")
        (dgrad,) = torch.autograd.grad(loss.sum(), z)
        results.append((*got, grad, loss, dgrad))
    for w, g in zip(*results):
        assert torch.equal(w, g)  # where a row lies changes nothing


def test_leading_dimensions(device):
    import k2_amd as k2
    x = orc.logits_case(9, 2 * 3 * 5, 120, torch.float32, device)
    tokens = torch.randint(0, 120, (30, 2), device=device)
    flat = k2.get_token_logprobs(x, tokens, num_top=3, return_entropy=True)
    deep = k2.get_token_logprobs(x.view(2, 3, 5, 120), tokens.view(2, 3, 5, 2), num_top=3, return_entropy=True)
    assert deep.logprobs.shape == (2, 3, 5, 2) and deep.entropy.shape == (2, 3, 5) and deep.top_tokens.shape == (2, 3, 5, 3)
    for f, d in zip(flat, deep):
        assert torch.equal(f, d.view(f.shape))
    permuted = x.view(2, 3, 5, 120).permute(2, 0, 1, 3)  # rows at no common distance: copied
    got = k2.get_token_logprobs(permuted, tokens.view(2, 3, 5, 2).permute(2, 0, 1, 3), num_top=3)
    assert torch.equal(got.logprobs, flat.logprobs.view(2, 3, 5, 2).permute(2, 0, 1, 3))
    one = k2.get_token_logprobs(x[4], tokens[4, 0], num_top=3)
    assert one.logprobs.shape == () and torch.equal(one.top_tokens, flat.top_tokens[4])
    same = k2.get_token_logprobs(x[4:5].expand(6, 120), tokens[4:5, 0].expand(6))  # stride 0 between rows
    assert torch.equal(same.logprobs, flat.logprobs[4, 0].expand(6))
    none = k2.get_token_logprobs(x[:0], tokens[:0], num_top=3, return_entropy=True)
    assert none.logprobs.shape == (0, 2) and none.top_tokens.shape == (0, 3)
    lone = x[4:5].clone().requires_grad_()
    many = lone.expand(6, 120)
    (grad,) = torch.autograd.grad(k2.get_token_logprobs(many, tokens[:6, 0]).logprobs.sum(), lone)
    wide = x[4:5].repeat(6, 1).requires_grad_()
    (want,) = torch.autograd.grad(k2.get_token_logprobs(wide, tokens[:6, 0]).logprobs.sum(), wide)
    torch.testing.assert_close(grad, want.sum(0, keepdim=True))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C,n,k", [(1, 1, 1), (6, 2, 6), (9, 1, 0), (65, 3, 4), (500, 1, 0), (500, 1, 8), (1237, 64, 64),
                                   (2049, 2, 20), (4999, 1, 0), (32001, 5, 33), (131072, 1, 0), (150001, 1, 10)])
def test_gradients_of_log_probs_entropy_and_alternatives(device, dtype, C, n, k):
    import k2_amd as k2
    rows = 9
    for temperature, use in ((1.0, "lht"), (0.5, "l"), (2.5, "h"), (1.0, "t")):
        if use == "t" and k == 0:
            continue
        x = orc.logits_case(C + n, rows, C, dtype, device).requires_grad_()
        gen = torch.Generator(device=device).manual_seed(7)
        tokens = torch.randint(0, C, (rows, n), generator=gen, device=device)
        tokens[2, 0] = -1
        if n > 1:
            tokens[3, 1] = tokens[3, 0]  # the same token twice
        tokens[4, 0] = C - 1
        mask = torch.ones(rows, dtype=torch.bool, device=device)
        mask[5] = False
        got = k2.get_token_logprobs(x, tokens, mask=mask, temperature=temperature, num_top=k, return_entropy=True)
        tokens_of = {"l": got.logprobs, "h": got.entropy, "t": got.top_logprobs}
        ups = {c: torch.randn(tokens_of[c].shape, generator=gen, device=device) for c in use if tokens_of[c] is not None}
        if "t" in ups:
            ups["t"][got.top_tokens < 0] = 0.0
        outputs = [tokens_of[c] for c in ups]
        (grad,) = torch.autograd.grad(outputs, x, [ups[c] for c in ups])
        orc.check_token_grad(x.detach(), tokens, mask, temperature,
                             (ups.get("l"), ups["h"].unsqueeze(1) if "h" in ups else None, ups.get("t")), got.top_tokens, grad)
        assert grad[5].eq(0).all()


@pytest.mark.parametrize("C", [5, 500, 4999, 131072])
def test_rows_of_nothing_get_no_gradient(device, C):
    """A row of nothing but -inf: log-probs that no logit moves, whatever is sent back through them."""
    import k2_amd as k2
    for dtype in DTYPES:
        x = orc.logits_case(C, 3, C, dtype, device)
        x[1] = NEG
        x.requires_grad_()
        got = k2.get_token_logprobs(x, torch.tensor([[0, C - 1]] * 3, device=device), num_top=2, return_entropy=True)
        ups = [torch.full_like(u, 3.0) for u in (got.logprobs, got.entropy, got.top_logprobs)]
        ups[0][1, 0] = float("inf")
        (grad,) = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], x, ups)
        assert grad[1].eq(0).all() and grad[0].ne(0).any() and grad[2].ne(0).any()


def test_gradients_against_differences(device):
    """Central differences of the operators themselves along random directions: f(x + h v) - f(x - h v) over 2 h.  The two
    values are each at most E off (the forward budgets: some 1e-5 for sums of a few rows) and the third derivative of a
    log-softmax along a unit direction is below 1, so the quotient is within E / h + h^2 of the derivative: h = 0.05."""
    import k2_amd as k2
    rows, C, h = 3, 40, 0.05
    x = orc.logits_case(2, rows, C, torch.float32, device, scale=0.7)
    a, t = orc.teacher_case(4, x, 6, 1.0)
    tokens = torch.randint(0, C, (rows,), device=device)

    def values(z):
        got = k2.get_token_logprobs(z, tokens, num_top=2, return_entropy=True)
        return [got.logprobs.sum(), got.entropy.sum(), got.top_logprobs.sum(),
                k2.distillation_loss(z, a, t, reduction="sum"), k2.distillation_loss(z, a, t, rest="bucket", reduction="sum")]

    z = x.clone().requires_grad_()
    grads = [torch.autograd.grad(f, z, retain_graph=True)[0] for f in values(z)]
    gen = torch.Generator(device=device).manual_seed(1)
    for _ in range(4):
        v = torch.randn(rows, C, generator=gen, device=device)
        v = v / v.norm()
        for i, (up, down) in enumerate(zip(values(x + h * v), values(x - h * v))):
            slope = (up - down).item() / (2 * h)
            assert abs(slope - (grads[i] * v).sum().item()) <= 6e-5 / h + 3 * h * h, i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bucket", [False, True])
@pytest.mark.parametrize("C,K", [(2, 1), (7, 7), (9, 3), (40, 64), (500, 4), (500, 8), (511, 17), (1237, 256), (2049, 20),
                                 (4999, 64), (32000, 20), (65537, 5), (131072, 64), (200001, 100)])
def test_distillation(device, dtype, bucket, C, K):
    import k2_amd as k2
    rows = 11
    for seed, temperature, holes, repeat, kept in ((0, 1.0, False, False, None), (1, 2.0, True, False, None),
                                                   (2, 0.7, False, True, 0.999), (3, 1.0, True, True, 0.5)):
        x = orc.logits_case(C + seed, rows, C, dtype, device).requires_grad_()
        a, t = orc.teacher_case(seed, x.detach(), K, temperature, holes, repeat, kept if K < C else None)
        mask = _mask(seed, rows, device) if seed % 2 else None
        gen = torch.Generator(device=device).manual_seed(seed)
        up = torch.randn(rows, generator=gen, device=device)
        loss = k2.distillation_loss(x, a, t, mask=mask, temperature=temperature, rest="bucket" if bucket else "renormalise",
                                    reduction="none")
        (grad,) = torch.autograd.grad(loss, x, up)
        orc.check_distillation(x.detach(), a, t, mask, temperature, bucket, loss, up, grad)


@pytest.mark.parametrize("bucket", [False, True])
def test_distillation_reductions(device, bucket):
    import k2_amd as k2
    rest = "bucket" if bucket else "renormalise"
    for rows in (1, 37, 9000, 20001):
        x = orc.logits_case(rows, rows, 60, torch.float32, device).requires_grad_()
        a, t = orc.teacher_case(1, x.detach(), 5, 1.0, holes=True)
        for mask in (None, _mask(rows, rows, device), torch.zeros(rows, dtype=torch.bool, device=device)):
            loss, err, grad, grad_err = orc.distillation(x.detach(), a, t, mask, 1.0, bucket)
            count = rows if mask is None else max(int(mask.sum()), 1)
            for reduction, divide in (("sum", 1), ("mean", count)):
                got = k2.distillation_loss(x, a, t, mask=mask, rest=rest, reduction=reduction)
                assert got.shape == ()
                want = loss.sum() / divide
                assert abs(got.double() - want) <= err.sum() / divide + 2 * orc.U * want.abs() + 1e-30
                (g,) = torch.autograd.grad(got * 0.3, x)
                orc.close("grad", g, grad * (0.3 / divide), grad_err * (0.3 / divide) + 4 * orc.U * grad.abs() * 0.3 / divide + 1e-37)


def test_student_with_nothing_outside_the_list(device):
    """bucket: a list of the whole vocabulary, a student that a mask keeps to the list, and one whose rest is far below
    what exp() can hold: the rest's own maximum keeps it."""
    import k2_amd as k2
    C = 6
    x = torch.tensor([[1.0, 2.0, 0.5, -1.0, 0.0, 3.0], [1.0, 2.0, NEG, NEG, NEG, NEG], [150.0, 149.0, -30.0, -31.0, -32.0, -33.0],
                      [NEG] * 6], device=device).requires_grad_()
    t = torch.tensor([[0, 1, 2, 3, 4, 5], [0, 1, -1, -1, -1, -1], [0, 1, -1, -1, -1, -1], [0, 1, -1, -1, -1, -1]], device=device)
    a = torch.full((4, 6), NEG, device=device)
    a[0] = torch.log_softmax(torch.arange(6.0, device=device), 0)
    a[1:, :2] = torch.tensor([0.5, 0.3], device=device).log()
    loss = k2.distillation_loss(x, a, t, rest="bucket", reduction="none")
    (grad,) = torch.autograd.grad(loss[:3], x, torch.ones(3, device=device))
    want, err, want_grad, grad_err = orc.distillation(x.detach()[:3], a[:3], t[:3], None, 1.0, True)
    orc.close("loss", loss[:3], want, err)
    orc.close("grad", grad[:3], want_grad, grad_err + 1e-30)
    assert want[2] > 30 and loss[3] == float("inf")
    for rest in ("renormalise", "bucket"):
        (grad,) = torch.autograd.grad(k2.distillation_loss(x, a, t, rest=rest, reduction="none")[3], x)
        assert torch.isfinite(grad[3]).all() and grad[3, 2:].eq(0).all() and grad[3, :2].lt(0).all()


def _lattice(device, dtype, B=3, T=40, S=12, R=4, C=70, seed=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    frames = torch.tensor([T, T - 7, T // 2][:B], device=device)
    ends = torch.tensor([S, S - 3, S // 2][:B], device=device)
    start = (torch.arange(T, device=device) * (S + 1 - R) // T).expand(B, T)
    ranges = (start.unsqueeze(2) + torch.arange(R, device=device)).contiguous()
    boundary = torch.zeros(B, 4, dtype=torch.int64, device=device)
    boundary[:, 2], boundary[:, 3] = ends, frames
    logits = orc.logits_case(seed, B * T * R, C, dtype, device).view(B, T, R, C)
    symbols = torch.randint(1, C, (B, S), generator=gen, device=device)
    inside = (torch.arange(T, device=device)[None, :, None] < frames[:, None, None]) & (ranges <= ends[:, None, None])
    return logits, ranges, boundary, symbols, inside


@pytest.mark.parametrize("dtype", DTYPES)
def test_pruned_lattice(device, dtype):
    import k2_amd as k2
    logits, ranges, boundary, _, inside = _lattice(device, dtype)
    assert torch.equal(k2.get_pruned_mask(ranges, boundary), inside)
    B, T, R, C = logits.shape
    logits[~inside] = float("nan")
    x = logits.clone().requires_grad_()
    a, t = orc.teacher_case(5, logits.view(-1, C), 6, 1.0)
    a, t = a.view(B, T, R, 6), t.view(B, T, R, 6)
    for rest in ("renormalise", "bucket"):
        want, err, want_grad, grad_err = orc.distillation(logits.view(-1, C), a.view(-1, 6), t.view(-1, 6), inside.view(-1), 1.0,
                                                          rest == "bucket")
        for reduction in ("none", "sum", "mean"):
            loss = k2.rnnt_distillation_loss_pruned(x, a, t, ranges, boundary, rest=rest, reduction=reduction)
            per = want.view(B, -1).sum(1)
            e = err.view(B, -1).sum(1)
            up = torch.tensor([0.5, -1.0, 2.0], device=device) if reduction == "none" else torch.tensor(0.5, device=device)
            divide = B if reduction == "mean" else 1
            if reduction != "none":
                per, e = per.sum() / divide, e.sum() / divide
            orc.close(reduction, loss, per, e + 4 * orc.U * per.abs())
            (grad,) = torch.autograd.grad(loss, x, up)
            ups = (up if reduction == "none" else up.expand(B) / divide).double().repeat_interleave(T * R).unsqueeze(1)
            w = want_grad * ups
            orc.close("grad", grad.view(-1, C), w, grad_err * ups.abs() + 4 * orc.U * w.abs() + orc._narrow(dtype, w))


@pytest.mark.parametrize("dtype", DTYPES)
def test_teacher_to_student_on_the_pruned_lattice(device, dtype):
    """As a recipe runs them: the teacher's logits are labelled on the pruned lattice, the student learns from the labels
    and from the transcript together."""
    import k2_amd as k2
    student, ranges, boundary, symbols, inside = _lattice(device, dtype, seed=1)
    teacher = _lattice(device, dtype, seed=2)[0]
    mask = k2.get_pruned_mask(ranges, boundary)
    tau, K = 2.0, 8
    with torch.no_grad():
        labels = k2.get_token_logprobs(teacher, mask=mask, temperature=tau, num_top=K)
    assert labels.top_tokens[~inside].eq(-1).all() and labels.top_logprobs[~inside].eq(NEG).all()
    x = student.clone().requires_grad_()
    pruned = k2.rnnt_loss_pruned(x.float(), symbols, ranges, 0, boundary, reduction="sum")
    distilled = k2.rnnt_distillation_loss_pruned(x, labels.top_logprobs, labels.top_tokens, ranges, boundary, temperature=tau,
                                                 rest="bucket", reduction="sum")
    (pruned + 0.25 * tau * tau * distilled).backward()
    y = student.clone().requires_grad_()
    (pruned_grad,) = torch.autograd.grad(k2.rnnt_loss_pruned(y.float(), symbols, ranges, 0, boundary, reduction="sum"), y)
    C = student.shape[-1]
    sm = orc.Softmax(teacher.reshape(-1, C), tau)
    order = orc.top(teacher.reshape(-1, C), K)
    exact_labels = sm.logp.gather(1, order)
    want, err, grad, grad_err = orc.distillation(student.reshape(-1, C), exact_labels.float(), order, inside.reshape(-1), tau, True)
    # (the labels' own error, at most 1e-5 each, moves the loss of a row by at most about that times (|log ratio| + 1) <= 20)
    live = inside.sum().item()
    assert abs(distilled.double() - want.sum()) <= err.sum() + 20e-5 * live * 1e-1 + 4 * orc.U * want.sum()
    total = pruned_grad.double().reshape(-1, C) + grad
    size = torch.finfo(dtype).eps
    torch.testing.assert_close(x.grad.double().reshape(-1, C), total, rtol=4 * size, atol=4 * size * 1.0 + 1e-4)


def test_two_runs_give_the_same_bits(device):
    import k2_amd as k2
    for dtype in DTYPES:
        for rows, C in ((3000, 500), (300, 33001)):
            x = orc.logits_case(1, rows, C, dtype, device).requires_grad_()
            a, t = orc.teacher_case(1, x.detach(), 12, 1.0, repeat=True)
            tokens = torch.randint(0, C, (rows, 3), device=device)
            results = []
            for _ in range(3):
                got = k2.get_token_logprobs(x, tokens, num_top=9, return_entropy=True)
                (g1,) = torch.autograd.grad([got.logprobs.sum(), got.entropy.sum(), got.top_logprobs.sum()], x)
                loss = k2.distillation_loss(x, a, t, rest="bucket")
                (g2,) = torch.autograd.grad(loss, x)
                results.append((*got, g1, loss, g2))
            for other in results[1:]:
                for u, v in zip(results[0], other):
                    assert torch.equal(u, v)


def test_on_another_stream_and_in_graphs(device):
    """On a side stream; captured twice and replayed in turn with new inputs, with eager work in between."""
    import k2_amd as k2
    rows, C, K = 130, 501, 6
    x = orc.logits_case(1, rows, C, torch.bfloat16, device)
    a, t = orc.teacher_case(2, x, K, 1.0)
    tokens = torch.randint(0, C, (rows,), device=device)
    mask = _mask(3, rows, device)

    def step(z):
        got = k2.get_token_logprobs(z, tokens, mask=mask, num_top=5, return_entropy=True)
        loss = k2.distillation_loss(z, a, t, mask=mask, rest="bucket")
        (grad,) = torch.autograd.grad([got.logprobs.sum(), got.entropy.sum(), loss], z)
        return (*got, loss, grad)

    want = [u.detach().clone() for u in step(x.clone().requires_grad_())]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x.clone().requires_grad_())
    torch.cuda.current_stream().wait_stream(side)
    for u, v in zip(want, got):
        assert torch.equal(u, v)
    graphs = []
    for _ in range(2):
        inputs = x.clone()
        with torch.cuda.stream(side):
            for _ in range(2):
                step(inputs.detach().requires_grad_())
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs = step(inputs.detach().requires_grad_())
        graphs.append((graph, inputs, outputs))
    for turn in range(4):
        for i, (graph, inputs, outputs) in enumerate(graphs):
            y = orc.logits_case(10 * turn + i, rows, C, torch.bfloat16, device)
            eager = [u.detach().clone() for u in step(y.clone().requires_grad_())]
            inputs.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            for u, v in zip(eager, outputs):
                assert torch.equal(u, v), (turn, i)


def test_more_than_two_to_the_31_logits(device):
    """Row offsets beyond 32 bits: 40000 rows of 65536 bfloat16 logits (5.2 GB), the last rows against the definition."""
    import k2_amd as k2
    rows, C = 40000, 65536
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device=device)
    pick = torch.tensor([0, 1, 32767, 32768, rows - 2, rows - 1], device=device)
    part = orc.logits_case(3, len(pick), C, torch.bfloat16, device)
    x[pick] = part
    x.requires_grad_()
    tokens = torch.randint(0, C, (rows,), device=device)
    got = k2.get_token_logprobs(x, tokens, num_top=3, return_entropy=True)
    orc.check_token_logprobs(part, tokens[pick].unsqueeze(1), None, 1.0, 3, k2.TokenLogprobs(*(u.detach()[pick] for u in got)))
    (grad,) = torch.autograd.grad(got.logprobs.sum(), x)
    orc.check_token_grad(part, tokens[pick].unsqueeze(1), None, 1.0, (torch.ones(len(pick), 1, device=device), None, None), None,
                         grad[pick])
    assert grad[20000].float().sum().abs() < 0.01
    del got, grad
    a, t = orc.teacher_case(4, part, 7, 1.0)
    A = torch.full((rows, 7), NEG, device=device)
    Tt = torch.full((rows, 7), -1, dtype=torch.int64, device=device)
    A[pick], Tt[pick] = a, t
    loss = k2.distillation_loss(x, A, Tt, rest="bucket", reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), x)
    orc.check_distillation(part, a, t, None, 1.0, True, loss.detach()[pick], torch.ones(len(pick), device=device), grad[pick])
    assert grad[20000].eq(0).all()


def test_both_host_layers_agree(device, monkeypatch):
    from k2_amd import capi, native
    import k2_amd as k2
    if native._ext is None:
        pytest.skip("the C++ host layer is not built")
    x = orc.logits_case(1, 40, 333, torch.float16, device)
    a, t = orc.teacher_case(2, x, 5, 1.0, holes=True)
    mask = _mask(1, 40, device)
    tokens = torch.randint(0, 333, (40, 2), device=device)
    ranges = torch.arange(3, device=device).repeat(2, 4, 1)
    boundary = torch.tensor([[0, 0, 1, 4], [0, 1, 2, 3]], device=device)

    def results():
        z = x.clone().requires_grad_()
        got = k2.get_token_logprobs(z, tokens, mask=mask, num_top=7, return_entropy=True)
        loss = k2.distillation_loss(z, a, t, mask=mask, rest="bucket")
        (grad,) = torch.autograd.grad([got.logprobs.sum(), got.entropy.sum(), got.top_logprobs[mask].sum(), loss], z)
        return (*got, loss, grad, k2.get_pruned_mask(ranges, boundary))

    cpp = results()
    monkeypatch.setattr(native, "_ext", None)
    assert capi.lib() is not None
    for u, v in zip(cpp, results()):
        assert torch.equal(u, v)


def test_refusals_on_the_device(device):
    import k2_amd as k2
    x = torch.randn(4, 9, device=device, requires_grad=True)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        k2.get_token_logprobs(x.double())
    with pytest.raises(RuntimeError, match="differentiat|does not require grad"):
        got = k2.get_token_logprobs(x, torch.zeros(4, dtype=torch.int64, device=device)).logprobs
        (g,) = torch.autograd.grad(got.sum(), x, create_graph=True)
        g.sum().backward()
    assert not math.isnan(float(k2.get_token_logprobs(x.detach(), torch.zeros(4, dtype=torch.int64)).logprobs.sum()))  # tokens move
