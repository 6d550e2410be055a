"""Calls of k2_amd/token_loss.py at the edges of what it takes, on the GPU: lists with values that are no log-probs, forward-mode
tangents, sums of as many rows as are served, lattices without rows, rows next to others,
rows of nothing, long lists on short rows, the longest rows and the most of them, rows in parts in
graphs, two threads."""
import pytest
import torch

import token_oracle as orc

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NEG, INF, NAN = float("-inf"), float("inf"), float("nan")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [40, 500, 1237, 5000, 40001])
def test_lists_that_hold_no_log_probs(device, dtype, C):
    """NaN or +inf at a listed token makes its row's loss and gradient NaN and no other's; at a token that is absent, and in a
    row that is masked out, it says nothing."""
    import k2_amd as k2
    rows, K = 9, 6
    x = orc.logits_case(C, rows, C, dtype, device).requires_grad_()
    a, t = orc.teacher_case(1, x.detach(), K, 1.0)
    a[0, 1] = NAN
    a[1] = NAN
    a[2, 3] = INF
    a[3, 0], t[3, 0] = NAN, -1
    a[4] = NAN
    a[5, 2] = NEG
    mask = torch.ones(rows, dtype=torch.bool, device=device)
    mask[4] = False
    wrong = torch.zeros_like(mask)
    wrong[:3] = True
    a0 = torch.where(t < 0, torch.full_like(a, NEG), a)
    for rest in ("renormalise", "bucket"):
        loss = k2.distillation_loss(x, a, t, mask=mask, rest=rest, reduction="none")
        (grad,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
        assert torch.equal(loss.isnan(), wrong)
        assert grad[wrong].isnan().all()
        keep = ~wrong
        orc.check_distillation(x.detach()[keep], a0[keep], t[keep], mask[keep], 1.0, rest == "bucket", loss.detach()[keep],
                               torch.ones(rows - 3, device=device), grad[keep])
        assert k2.distillation_loss(x, a, t, mask=mask, rest=rest).isnan()
    teacher = x.detach().clone()
    teacher[6, 5] = INF
    labels = k2.get_token_logprobs(teacher, num_top=4)
    loss = k2.distillation_loss(x, labels.top_logprobs, labels.top_tokens, reduction="none")
    assert loss[6].isnan() and int(loss.isnan().sum()) == 1


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(device, requires_grad):
    """A tangent is never dropped, whether or not a gradient is asked for besides."""
    import k2_amd as k2
    import torch.autograd.forward_ad as fw
    x = torch.randn(3, 9, device=device).requires_grad_(requires_grad)
    a, t = torch.full((3, 2), -1.0, device=device), torch.tensor([[1, 2]] * 3, device=device)
    with fw.dual_level():
        dual, listed = fw.make_dual(x, torch.ones(3, 9, device=device)), fw.make_dual(a, torch.ones(3, 2, device=device))
        for call in (lambda: k2.get_token_logprobs(dual, num_top=2), lambda: k2.distillation_loss(dual, a, t),
                     lambda: k2.distillation_loss(x, listed, t)):
            with pytest.raises(NotImplementedError):
                call()


@pytest.mark.parametrize("rows", [(1 << 31) - 1, (1 << 31) - 1000, (1 << 31) - 2048])
def test_sum_of_as_many_rows_as_are_served(device, rows):
    """The losses next to the 2^31st row: the whole numbers here add up exactly, in double, to far less than 2^24."""
    from k2_amd import native
    losses = torch.zeros(rows, device=device)
    at = torch.tensor([0, 2047, 2048, 16384, 1 << 30, rows - 2500, rows - 2049, rows - 2048, rows - 1048, rows - 2, rows - 1], device=device)
    losses[at] = torch.arange(1.0, 12.0, device=device)
    total, _ = native.distillation_sum(losses, None, 1, False, 0.5)
    assert total.item() == 33.0
    mask = torch.zeros(rows, dtype=torch.bool, device=device)
    mask[at] = True
    mean, inverse = native.distillation_sum(losses, mask, 1, True, 1.0)
    assert mean.item() == 6.0 and inverse.item() == torch.tensor(1.0 / 11).item()


@pytest.mark.parametrize("B,T", [(0, 4), (2, 0)])
def test_lattices_without_rows(device, B, T):
    """One loss a sequence, however many sequences and rows of each there are."""
    import k2_amd as k2
    x = torch.zeros(B, T, 3, 9, device=device, requires_grad=True)
    a, t = torch.zeros(B, T, 3, 2, device=device), torch.zeros(B, T, 3, 2, dtype=torch.int64, device=device)
    ranges, boundary = torch.zeros(B, T, 3, dtype=torch.int64, device=device), torch.zeros(B, 4, dtype=torch.int64, device=device)
    for reduction in ("none", "sum", "mean"):
        loss = k2.rnnt_distillation_loss_pruned(x, a, t, ranges, boundary, reduction=reduction)
        assert loss.shape == ((B,) if reduction == "none" else ()) and loss.eq(0).all()
        assert torch.autograd.grad(loss, x, torch.ones_like(loss))[0].shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [9, 37, 300, 500, 1000, 1237])
def test_rows_do_not_see_their_neighbours(device, dtype, C):
    """Short rows share a wavefront: whatever the others hold, masked out or not, a row's bits are the same, and the same at
    every place in the batch."""
    import k2_amd as k2
    rows = 64
    x = orc.logits_case(C, rows, C, dtype, device)
    if dtype != torch.float16:
        x[6] = 3.0e7 * torch.sign(x[6].float()).to(dtype)  # (one that takes differences first)
    a, t = orc.teacher_case(1, x, 4, 1.0, repeat=True)
    gen = torch.Generator(device=device).manual_seed(C)
    keep = torch.rand(rows, generator=gen, device=device) < 0.4
    keep[6] = True
    others = torch.randn(int((~keep).sum()), C, generator=gen, device=device)
    fillings = [others, others * 1e4, others * 1e30, torch.full_like(others, torch.finfo(dtype).min),
                torch.full_like(others, NAN), torch.full_like(others, NEG), torch.full_like(others, INF)]

    def results(y, mask, a=a, t=t):
        y = y.requires_grad_()
        got = k2.get_token_logprobs(y, t[:, 0].clamp(min=0), mask=mask, num_top=3, return_entropy=True)
        (grad,) = torch.autograd.grad([got.logprobs, got.entropy], y, [torch.ones(len(y), device=device)] * 2)
        out = [*got, grad]
        for rest in ("renormalise", "bucket"):
            loss = k2.distillation_loss(y, a, t, mask=mask, rest=rest, reduction="none")
            out += [loss, torch.autograd.grad(loss.sum(), y)[0]]
        return [u.detach() for u in out]

    want = [u[keep] for u in results(x.clone(), None)]
    for mask in (keep, None):
        for filling in fillings:
            y = x.clone()
            y[~keep] = filling.to(dtype)
            for u, w in zip(results(y, mask), want):
                assert torch.equal(u[keep], w)
    order = torch.randperm(rows, generator=gen, device=device)
    for u, w in zip(results(x[order].clone(), None, a[order], t[order]), results(x.clone(), None)):
        assert torch.equal(u, w[order])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [5, 500, 1237, 4999, 131072])
def test_rows_of_nothing_whatever_is_sent_back(device, dtype, C):
    """A row of nothing but -inf has gradient 0, and a token past the vocabulary shows in it all the same."""
    import k2_amd as k2
    x = orc.logits_case(C, 4, C, dtype, device)
    x[1:3] = NEG
    x.requires_grad_()
    tokens = torch.tensor([[0, C - 1]] * 4, device=device)
    tokens[2, 1] = C
    got = k2.get_token_logprobs(x, tokens, num_top=2, return_entropy=True)
    for up in ([NAN, 0.0], [INF, NEG], [INF, INF], [1.0, NAN]):
        ups = [torch.full_like(u, 3.0) for u in (got.logprobs, got.entropy, got.top_logprobs)]
        for u in ups[0], ups[2]:
            u[1] = torch.tensor(up, device=device)
        ups[1][1] = up[0]
        (grad,) = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], x, ups, retain_graph=True)
        assert grad[1].eq(0).all() and grad[2].isnan().all() and torch.isfinite(grad[[0, 3]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [70, 300, 500, 512, 1000, 1024])
def test_long_lists_on_short_rows(device, dtype, C):
    """The most that a gradient keeps in LDS beside the rows it stages: 256 entries a row of a teacher's list, 64 given tokens
    and 64 alternatives."""
    import k2_amd as k2
    rows = 37
    for K in (65, 100, 256):
        x = orc.logits_case(C + K, rows, C, dtype, device).requires_grad_()
        a, t = orc.teacher_case(K, x.detach(), K, 1.0, holes=True, repeat=True)
        mask = torch.rand(rows, device=device) < 0.8
        up = torch.randn(rows, device=device)
        for bucket in (False, True):
            loss = k2.distillation_loss(x, a, t, mask=mask, rest="bucket" if bucket else "renormalise", reduction="none")
            (grad,) = torch.autograd.grad(loss, x, up)
            orc.check_distillation(x.detach(), a, t, mask, 1.0, bucket, loss, up, grad)
    for n, k in ((17, 0), (3, 20), (64, 64)):
        x = orc.logits_case(C + n, rows, C, dtype, device).requires_grad_()
        tokens = torch.randint(0, C, (rows, n), device=device)
        tokens[1, 0], tokens[2, 1] = -1, tokens[2, 0]
        got = k2.get_token_logprobs(x, tokens, mask=mask, num_top=k, return_entropy=True)
        orc.check_token_logprobs(x.detach(), tokens, mask, 1.0, k,
                                 k2.TokenLogprobs(*(None if u is None else u.detach() for u in got)))
        ups = [torch.randn(rows, n, device=device), torch.randn(rows, device=device), torch.randn(rows, k, device=device) if k else None]
        (grad,) = torch.autograd.grad([u for u in (got.logprobs, got.entropy, got.top_logprobs) if u is not None], x,
                                      [u for u in ups if u is not None])
        if k:
            ups[2][got.top_tokens < 0] = 0.0
        orc.check_token_grad(x.detach(), tokens, mask, 1.0, (ups[0], ups[1].unsqueeze(1), ups[2]), got.top_tokens, grad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [(1 << 20) - 3, 1 << 20])
@pytest.mark.parametrize("rows", [1, 3, 300])
def test_the_longest_rows(device, dtype, C, rows):
    """Rows of as many columns as are served, in up to 64 parts."""
    import k2_amd as k2
    pick = torch.arange(rows, device=device)[-2:]
    x = orc.logits_case(rows, rows, C, dtype, device).requires_grad_()
    tokens = torch.randint(0, C, (rows, 1), device=device)
    tokens[-1] = C - 1
    got = k2.get_token_logprobs(x, tokens, num_top=64, return_entropy=True)
    orc.check_token_logprobs(x.detach()[pick], tokens[pick], None, 1.0, 64, k2.TokenLogprobs(*(u.detach()[pick] for u in got)))
    ups = torch.randn(rows, 1, device=device), torch.randn(rows, device=device), torch.randn(rows, 64, device=device)
    (grad,) = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], x, ups)
    orc.check_token_grad(x.detach()[pick], tokens[pick], None, 1.0, (ups[0][pick], ups[1][pick].unsqueeze(1), ups[2][pick]),
                         got.top_tokens[pick], grad[pick])
    without = k2.get_token_logprobs(x.detach(), tokens, return_entropy=True)
    orc.check_token_logprobs(x.detach()[pick], tokens[pick], None, 1.0, 0,
                             k2.TokenLogprobs(without.logprobs[pick], without.entropy[pick], None, None))
    del got, grad, without
    a, t = orc.teacher_case(1, x.detach()[pick], 100, 1.0, repeat=True)
    A, Tt = torch.full((rows, 100), NEG, device=device), torch.full((rows, 100), -1, dtype=torch.int64, device=device)
    A[pick], Tt[pick] = a, t
    up = torch.randn(rows, device=device)
    for rest in ("renormalise", "bucket"):
        loss = k2.distillation_loss(x, A, Tt, rest=rest, reduction="none")
        (grad,) = torch.autograd.grad(loss, x, up)
        orc.check_distillation(x.detach()[pick], a, t, None, 1.0, rest == "bucket", loss.detach()[pick], up[pick], grad[pick])


def test_more_long_rows_than_a_launch_takes(device):
    """Rows of several wavefronts beyond 2^20 of them: the last rows of both launches against the definition."""
    import k2_amd as k2
    rows, C = (1 << 20) + 5, 2056
    pick = torch.tensor([0, (1 << 20) - 1, 1 << 20, rows - 1], device=device)
    part = orc.logits_case(3, len(pick), C, torch.bfloat16, device)
    x = torch.zeros(rows, C, dtype=torch.bfloat16, device=device)
    x[pick] = part
    x.requires_grad_()
    tokens = torch.randint(0, C, (rows,), device=device)
    mask = torch.ones(rows, dtype=torch.bool, device=device)
    mask[(1 << 20) + 1] = False
    for k in (0, 2):
        got = k2.get_token_logprobs(x, tokens, mask=mask, num_top=k, return_entropy=True)
        orc.check_token_logprobs(part, tokens[pick].unsqueeze(1), None, 1.0, k,
                                 k2.TokenLogprobs(*(None if u is None else u.detach()[pick] for u in got)))
        assert got.logprobs[(1 << 20) + 1] == 0 and got.entropy[(1 << 20) + 1] == 0
    (grad,) = torch.autograd.grad(got.logprobs.sum(), x)
    orc.check_token_grad(part, tokens[pick].unsqueeze(1), None, 1.0, (torch.ones(len(pick), 1, device=device), None, None), None,
                         grad[pick])
    assert grad[(1 << 20) + 1].eq(0).all()
    del grad, got
    a, t = orc.teacher_case(4, part, 3, 1.0)
    A, Tt = torch.full((rows, 3), NEG, device=device), torch.full((rows, 3), -1, dtype=torch.int64, device=device)
    A[pick], Tt[pick] = a, t
    loss = k2.distillation_loss(x, A, Tt, mask=mask, rest="bucket", reduction="none")
    (grad,) = torch.autograd.grad(loss.sum(), x)
    orc.check_distillation(part, a, t, None, 1.0, True, loss.detach()[pick], torch.ones(len(pick), device=device), grad[pick])
    assert int(grad.ne(0).any(1).sum()) == len(pick) and int(loss.ne(0).sum()) == len(pick)


def test_rows_in_parts_in_graphs(device):
    """Calls that join parts of rows through scratch memory, captured twice and replayed in turn with new inputs."""
    import k2_amd as k2
    rows, C, K = 5, 40009, 6
    x = orc.logits_case(1, rows, C, torch.float32, device)
    a, t = orc.teacher_case(2, x, K, 1.0)
    tokens = torch.randint(0, C, (rows,), device=device)
    mask = torch.tensor([True, True, False, True, True], device=device)

    def step(z):
        got = k2.get_token_logprobs(z, tokens, mask=mask, num_top=9, return_entropy=True)
        plain = k2.get_token_logprobs(z, tokens, mask=mask)
        loss = k2.distillation_loss(z, a, t, mask=mask, rest="bucket")
        (grad,) = torch.autograd.grad([got.logprobs.sum(), got.entropy.sum(), plain.logprobs.sum(), loss], z)
        return (*got, plain.logprobs, loss, grad)

    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        inputs = x.clone()
        side.wait_stream(torch.cuda.current_stream())
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
            y = orc.logits_case(10 * turn + i, rows, C, torch.float32, device)
            eager = [u.detach().clone() for u in step(y.clone().requires_grad_())]
            inputs.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            for u, v in zip(eager, outputs):
                assert torch.equal(u, v), (turn, i)


def test_calls_from_two_threads_on_two_streams(device):
    """The host layers hold no lock and no workspace: forward and backward at once on streams of their own."""
    import threading
    import k2_amd as k2
    rows, C = 64, 33001
    x = [orc.logits_case(i, rows, C, torch.bfloat16, device) for i in range(2)]
    lists = [orc.teacher_case(i, x[i], 5, 1.0) for i in range(2)]
    torch.cuda.synchronize()

    def step(i):
        z = x[i].detach().requires_grad_()
        got = k2.get_token_logprobs(z, lists[i][1][:, 0], num_top=9, return_entropy=True)
        loss = k2.distillation_loss(z, *lists[i], rest="bucket", reduction="sum")
        (grad,) = torch.autograd.grad([got.logprobs.sum(), got.entropy.sum(), loss], z)
        return [u.detach() for u in (*got, loss, grad)]

    want, failures = [step(0), step(1)], []
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = step(i)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(u, v) for u, v in zip(got, want[i]))
        except BaseException as error:  # (a thread's failure is not the test's by itself)
            failures.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures
