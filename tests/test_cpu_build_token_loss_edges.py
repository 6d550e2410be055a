"""Calls of k2_amd/token_loss.py at the edges of what it takes, on the host build of the kernels through both host layers: lists
with values that are no log-probs, forward-mode tangents, lattices without rows, rows next to others,
rows of nothing, tensors marked as negated, long lists on short rows."""
import pytest
import torch

import token_oracle as orc
from test_cpu_build_host_layer import host_on_cpu  # noqa: F401  (a fixture)
from test_cpu_build_token_loss import host  # noqa: F401  (a fixture)

CPU = torch.device("cpu")
NEG, INF, NAN = float("-inf"), float("inf"), float("nan")


def _lists_that_hold_no_log_probs(C, dtype, rests):
    import k2_amd as k2
    x = orc.logits_case(C, 7, C, dtype, CPU).requires_grad_()
    a, t = orc.teacher_case(1, x.detach(), 4, 1.0)
    a[0, 1] = NAN
    a[1] = NAN
    a[2, 3] = INF
    a[3, 0], t[3, 0] = NAN, -1
    a[4] = NAN
    a[5, 2] = NEG
    mask = torch.tensor([True, True, True, True, False, True, True])
    wrong = torch.tensor([True, True, True, False, False, False, False])
    for rest in rests:
        loss = k2.distillation_loss(x, a, t, mask=mask, rest=rest, reduction="none")
        (grad,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
        assert torch.equal(loss.isnan(), wrong), loss
        assert grad[wrong].isnan().all() and torch.isfinite(grad[~wrong]).all()
        a0 = torch.where(t < 0, torch.full_like(a, NEG), a)
        orc.check_distillation(x.detach()[~wrong], a0[~wrong], t[~wrong], mask[~wrong], 1.0, rest == "bucket", loss.detach()[~wrong],
                               torch.ones(4), grad[~wrong])
    return x.detach(), a, t, mask


def test_lists_that_hold_no_log_probs(host):  # noqa: F811
    """NaN or +inf at a listed token makes its row's loss and gradient NaN and no other's; at a token that is absent, and in a
    row that is masked out, it says nothing.  -inf is probability 0."""
    import k2_amd as k2
    rests = ("renormalise", "bucket")
    x, a, t, mask = _lists_that_hold_no_log_probs(40, torch.float32, rests)
    for rest in rests:
        for reduction in ("sum", "mean"):
            assert k2.distillation_loss(x, a, t, mask=mask, rest=rest, reduction=reduction).isnan()
    # from a teacher's row that overflowed, as its labelling lists it
    x[6, 5] = INF
    labels = k2.get_token_logprobs(x, num_top=4)
    assert labels.top_tokens[6].ge(0).all()
    loss = k2.distillation_loss(x[:1].expand(7, 40), labels.top_logprobs, labels.top_tokens, reduction="none")
    assert loss[6].isnan() and torch.isfinite(loss[:6]).all()


# (rows that wavefronts read along; rows in two parts)
@pytest.mark.parametrize("C,dtype,rest", [(700, torch.bfloat16, "renormalise"), (1100, torch.float32, "bucket"),
                                          (1100, torch.float32, "renormalise"), (4200, torch.float32, "bucket")])
def test_lists_that_hold_no_log_probs_of_long_rows(host_on_cpu, C, dtype, rest):  # noqa: F811
    _lists_that_hold_no_log_probs(C, dtype, (rest,))


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_forward_mode_is_refused(host, requires_grad, grad_mode):  # noqa: F811
    """A tangent is never dropped: with or without a gradient besides, in logits and in the teacher's log-probs."""
    import k2_amd as k2
    import torch.autograd.forward_ad as fw
    x = torch.randn(3, 9).requires_grad_(requires_grad)
    tokens, a, t = torch.zeros(3, dtype=torch.int64), torch.full((3, 2), -1.0), torch.tensor([[1, 2]] * 3)
    lattice = (torch.arange(3).reshape(1, 1, 3), torch.tensor([[0, 0, 2, 1]]))
    with torch.set_grad_enabled(grad_mode), fw.dual_level():
        dual = fw.make_dual(x, torch.ones(3, 9))
        listed = fw.make_dual(a, torch.ones(3, 2))
        for call in (lambda: k2.get_token_logprobs(dual, tokens), lambda: k2.get_token_logprobs(dual, return_entropy=True, num_top=2),
                     lambda: k2.distillation_loss(dual, a, t), lambda: k2.distillation_loss(x, listed, t, reduction="none"),
                     lambda: k2.rnnt_distillation_loss_pruned(dual.view(1, 1, 3, 9), a.view(1, 1, 3, 2), t.view(1, 1, 3, 2), *lattice)):
            with pytest.raises(NotImplementedError):
                call()
        # the primal alone is as good as any tensor, and so is a level that nothing was made dual in
        assert torch.equal(k2.get_token_logprobs(fw.unpack_dual(dual).primal, tokens).logprobs,
                           k2.get_token_logprobs(x, tokens).logprobs)
    assert k2.get_token_logprobs(x, tokens).logprobs.requires_grad == requires_grad


@pytest.mark.parametrize("B,T,R", [(0, 4, 3), (2, 0, 3), (0, 0, 3)])
def test_lattices_without_rows(host, B, T, R):  # noqa: F811
    """One loss a sequence, however many sequences and rows of each there are."""
    import k2_amd as k2
    x = torch.zeros(B, T, R, 9, requires_grad=True)
    a, t = torch.zeros(B, T, R, 2), torch.zeros(B, T, R, 2, dtype=torch.int64)
    ranges, boundary = torch.zeros(B, T, R, dtype=torch.int64), torch.zeros(B, 4, dtype=torch.int64)
    for box in (None, boundary):
        for logits in (x, x.detach()):
            for reduction in ("none", "sum", "mean"):
                loss = k2.rnnt_distillation_loss_pruned(logits, a, t, ranges, box, reduction=reduction)
                assert loss.shape == ((B,) if reduction == "none" else ()) and loss.eq(0).all()
                assert loss.requires_grad == logits.requires_grad
                if logits.requires_grad:
                    (grad,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
                    assert grad.shape == x.shape
    assert k2.distillation_loss(x, a, t, reduction="none").shape == (B, T, R)


@pytest.mark.parametrize("C,dtype", [(37, torch.float32), (300, torch.bfloat16)])
def test_rows_do_not_see_their_neighbours(host, C, dtype):  # noqa: F811
    """Four short rows share a wavefront: whatever three of them hold, masked out or not, the fourth's bits are the same."""
    import k2_amd as k2
    rows = 8
    x = orc.logits_case(C, rows, C, dtype, CPU)
    x[6] = 3.0e7 * torch.sign(x[6].float()).to(dtype)  # (one that takes differences first)
    a, t = orc.teacher_case(1, x, 4, 1.0, repeat=True)
    keep = torch.tensor([True, False, False, True, False, False, True, False])
    others = torch.randn(int((~keep).sum()), C)
    fillings = [others, others * 1e30, torch.full_like(others, NAN), torch.full_like(others, INF)]
    for mask in (keep, None) if C == 37 else (None,):
        want = None
        for filling in fillings:
            y = x.clone()
            y[~keep] = filling.to(dtype)
            y.requires_grad_()
            got = k2.get_token_logprobs(y, t[:, 0].clamp(min=0), mask=mask, num_top=3, return_entropy=True)
            (grad,) = torch.autograd.grad([got.logprobs, got.entropy], y, [torch.ones(rows)] * 2)
            results = [*got, grad]
            for rest in ("renormalise", "bucket"):
                loss = k2.distillation_loss(y, a, t, mask=mask, rest=rest, reduction="none")
                results += [loss, torch.autograd.grad(loss.sum(), y)[0]]
            results = [u.detach()[keep] for u in results]
            want = want or results
            for u, w in zip(results, want):
                assert torch.equal(u, w)


@pytest.mark.parametrize("C,dtype,up", [(1, torch.float32, [NAN, 0.0]), (40, torch.bfloat16, [INF, NEG]), (40, torch.float32, [INF, INF]),
                                        (40, torch.float16, [1.0, NAN]), (700, torch.float32, [NAN, 0.0]),
                                        (2300, torch.float16, [INF, NEG])])
def test_rows_of_nothing_whatever_is_sent_back(host, C, dtype, up):  # noqa: F811
    """A row of nothing but -inf has gradient 0, and a token past the vocabulary shows in it all the same."""
    import k2_amd as k2
    x = orc.logits_case(C, 4, C, dtype, CPU)
    x[1:3] = NEG
    x.requires_grad_()
    tokens = torch.tensor([[0, C - 1]] * 4)
    tokens[2, 1] = C
    got = k2.get_token_logprobs(x, tokens, num_top=2, return_entropy=True)
    ups = [torch.full_like(u, 3.0) for u in (got.logprobs, got.entropy, got.top_logprobs)]
    for u in ups[0], ups[2]:
        u[1] = torch.tensor(up)
    ups[1][1] = up[0]
    (grad,) = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], x, ups, retain_graph=True)
    assert grad[1].eq(0).all() and grad[2].isnan().all() and torch.isfinite(grad[[0, 3]]).all()
    (grad,) = torch.autograd.grad(got.logprobs, x, ups[0])
    assert grad[1].eq(0).all() and grad[2].isnan().all()


def test_tensors_that_are_marked_as_negated(host):  # noqa: F811
    """torch hands out views whose memory holds the opposite sign (the imaginary part of a conjugate, say)."""
    import k2_amd as k2
    C = 21
    x = orc.logits_case(1, 5, C, torch.float32, CPU)
    a, t = orc.teacher_case(1, x, 3, 1.0)
    wide = torch.cat([-x, torch.full((5, 4), 99.0)], 1)
    up = torch.randn(5)

    def results(x, a, up):
        x = x.detach().requires_grad_()
        got = k2.get_token_logprobs(x, t[:, 0], num_top=2, return_entropy=True)
        loss = k2.distillation_loss(x, a, t, rest="bucket", reduction="none")
        return [*got, *torch.autograd.grad([got.logprobs, got.entropy], x, [up, up]), loss, *torch.autograd.grad(loss, x, up)]

    want = results(x, a, up)
    for args in ((torch._neg_view(-x), a, up), (torch._neg_view(wide)[:, :C], a, up), (x, torch._neg_view(-a), up),
                 (x, a, torch._neg_view(-up))):
        for u, w in zip(results(*args), want):
            assert torch.equal(u, w)


def test_long_lists_on_short_rows(host):  # noqa: F811
    """The most that a gradient keeps in LDS beside the rows it stages."""
    import k2_amd as k2
    C, rows, K = 300, 3, 256
    x = orc.logits_case(1, rows, C, torch.float32, CPU).requires_grad_()
    a, t = orc.teacher_case(1, x.detach(), K, 1.0, repeat=True)
    for bucket in (False, True):
        loss = k2.distillation_loss(x, a, t, rest="bucket" if bucket else "renormalise", reduction="none")
        (grad,) = torch.autograd.grad(loss, x, torch.ones(rows))
        orc.check_distillation(x.detach(), a, t, None, 1.0, bucket, loss.detach(), torch.ones(rows), grad)
    tokens = torch.randint(0, C, (rows, 64))
    got = k2.get_token_logprobs(x, tokens, num_top=64)
    ups = torch.randn(rows, 64), torch.randn(rows, 64)
    (grad,) = torch.autograd.grad([got.logprobs, got.top_logprobs], x, ups)
    orc.check_token_grad(x.detach(), tokens, None, 1.0, (ups[0], None, ups[1]), got.top_tokens, grad)
