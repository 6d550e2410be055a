"""The operators of k2_amd/token_loss.py on the host build of their kernels (tests/cpu_kernels.py), through both host
layers, against the definitions in 64 bits (tests/token_oracle.py); their C-ABI on fenced buffers; their refusals."""
import numpy as np
import pytest
import torch

import cpu_kernels as ck
import token_oracle as orc
from cpu_kernels import Fenced, fenced, p
from test_cpu_build_cpp_host_layer import hosts  # noqa: F401  (a fixture)
from test_cpu_build_host_layer import host_on_cpu  # noqa: F401  (a fixture)

CPU = torch.device("cpu")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
NEG = float("-inf")


@pytest.fixture(params=["ctypes", "c++"])
def host(request, host_on_cpu, monkeypatch):  # noqa: F811
    if request.param == "c++":
        from k2_amd import native
        monkeypatch.setattr(native, "_ext", ck.host_layer())
    return request.param


def _types_over(sizes):
    """Every size in one type, every type in one size."""
    return [(s, DTYPES[i % 3]) for i, s in enumerate(sizes)] + [(sizes[-2], d) for d in DTYPES if d != DTYPES[(len(sizes) - 2) % 3]]


@pytest.mark.parametrize("case,dtype", _types_over([(1, 1, 1), (7, 2, 9), (65, 1, 0), (300, 3, 20), (701, 1, 64)]))
def test_token_logprobs(host, case, dtype):
    import k2_amd as k2
    (C, n, k), rows = case, 5
    x = orc.logits_case(C, rows, C, dtype, CPU)
    if C > 4:
        x[1, 1:] = NEG
        x[2] = torch.finfo(dtype).min
        x[3] = 1.0
    x.requires_grad_()
    tokens = torch.randint(0, C, (rows, n))
    tokens[0, 0] = -1
    if n > 1:
        tokens[4, 1] = tokens[4, 0]
    mask = torch.tensor([True, True, True, True, False]) if k else None
    got = k2.get_token_logprobs(x, tokens, mask=mask, temperature=1.5, num_top=k, return_entropy=True)
    orc.check_token_logprobs(x.detach(), tokens, mask, 1.5, k, k2.TokenLogprobs(*(None if u is None else u.detach() for u in got)))
    ups = [torch.randn(rows, n), torch.randn(rows), torch.randn(rows, k) if k else None]
    tops = got.top_tokens
    outputs = [got.logprobs, got.entropy] + ([got.top_logprobs] if k else [])
    (grad,) = torch.autograd.grad(outputs, x, [u for u in ups if u is not None])
    orc.check_token_grad(x.detach(), tokens, mask, 1.5, (ups[0], ups[1].unsqueeze(1), ups[2]), tops, grad)


@pytest.mark.parametrize("bucket", [False, True])
@pytest.mark.parametrize("case,dtype", _types_over([(2, 1), (9, 9), (130, 5), (601, 33)]))
def test_distillation(host, case, dtype, bucket):
    import k2_amd as k2
    (C, K), rows = case, 6
    x = orc.logits_case(C, rows, C, dtype, CPU)
    a, t = orc.teacher_case(C, x, K, 2.0, holes=K > 3, repeat=K > 3)
    x.requires_grad_()
    mask = torch.tensor([True, True, False, True, True, True])
    up = torch.randn(rows)
    loss = k2.distillation_loss(x, a, t, mask=mask, temperature=2.0, rest="bucket" if bucket else "renormalise", reduction="none")
    (grad,) = torch.autograd.grad(loss, x, up)
    orc.check_distillation(x.detach(), a, t, mask, 2.0, bucket, loss.detach(), up, grad)
    mean = k2.distillation_loss(x, a, t, mask=mask, temperature=2.0, rest="bucket" if bucket else "renormalise")
    torch.testing.assert_close(mean.detach(), loss.detach().sum() / 5, rtol=1e-6, atol=1e-7)


def test_pruned_lattice(host):
    import k2_amd as k2
    B, T, R, C = 2, 6, 3, 20
    ranges = ((torch.arange(T) // 2).unsqueeze(1) + torch.arange(R)).expand(B, T, R).contiguous()
    boundary = torch.tensor([[0, 0, 4, 6], [1, 2, 3, 5]])
    t = torch.arange(T)[None, :, None]
    box = boundary[:, None, None, :]
    want = (t >= box[..., 1]) & (t < box[..., 3]) & (ranges >= box[..., 0]) & (ranges <= box[..., 2])
    assert torch.equal(k2.get_pruned_mask(ranges, boundary), want)
    x = orc.logits_case(1, B * T * R, C, torch.float32, CPU).view(B, T, R, C)
    a, tk = orc.teacher_case(1, x.view(-1, C), 4, 1.0)
    a, tk = a.view(B, T, R, 4), tk.view(B, T, R, 4)
    x[~want] = float("nan")
    x.requires_grad_()
    loss, err, grad, grad_err = orc.distillation(x.detach().view(-1, C), a.view(-1, 4), tk.view(-1, 4), want.view(-1), 1.0, True)
    for reduction in ("none", "sum", "mean"):
        got = k2.rnnt_distillation_loss_pruned(x, a, tk, ranges, boundary, rest="bucket", reduction=reduction)
        per, e = loss.view(B, -1).sum(1), err.view(B, -1).sum(1)
        d = B if reduction == "mean" else 1
        if reduction != "none":
            per, e = per.sum() / d, e.sum() / d
        orc.close(reduction, got.detach(), per, e + 4 * orc.U * per.abs())
        (g,) = torch.autograd.grad(got.sum(), x)
        orc.close("grad", g.view(-1, C), grad / d, grad_err / d + 4 * orc.U * grad.abs() + 1e-37)


def test_strides_and_empty_batches(host):
    import k2_amd as k2
    base = orc.logits_case(1, 12, 47, torch.bfloat16, CPU)
    tokens = torch.randint(0, 41, (12,))
    dense = base[:, :41].contiguous()
    want = k2.get_token_logprobs(dense, tokens, num_top=4, return_entropy=True)
    for view, tk in ((base[:, :41], tokens), (base[:, :41].view(3, 4, 41), tokens.view(3, 4)),
                     (dense.t().contiguous().t(), tokens), (dense.view(3, 4, 41).transpose(0, 1), tokens.view(3, 4).t())):
        got = k2.get_token_logprobs(view, tk, num_top=4, return_entropy=True)
        if view.dim() == 3 and view.shape[0] == 4:
            got = [u.transpose(0, 1).reshape(w.shape) for u, w in zip(got, want)]
        for u, w in zip(got, want):
            assert torch.equal(u.reshape(w.shape), w)
    none = k2.get_token_logprobs(dense[:0], tokens[:0], num_top=2, return_entropy=True)
    assert none.top_tokens.shape == (0, 2) and none.entropy.shape == (0,)
    x = dense[:0].detach().requires_grad_()
    for reduction in ("none", "sum", "mean"):
        loss = k2.distillation_loss(x, torch.zeros(0, 3), torch.zeros(0, 3, dtype=torch.int64), reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and loss.sum() == 0
        assert torch.autograd.grad(loss.sum(), x)[0].shape == (0, 41)


@pytest.fixture(scope="module")
def lib():
    return ck.lib()


@pytest.mark.parametrize("at,dtype,code,C", [
    ("end", np.float32, 0, 1), ("end", np.uint16, 3, 3), ("start", np.uint16, 2, 7), ("end", np.uint16, 3, 8),
    ("end", np.float32, 0, 61), ("start", np.float32, 0, 61), ("end", np.uint16, 2, 515), ("start", np.uint16, 3, 515),
    # several wavefronts a row; rows in parts
    ("end", np.float32, 0, 1031), ("end", np.uint16, 3, 8203), ("end", np.float32, 0, 8197)])
def test_nothing_outside_the_tensors_is_touched(lib, at, dtype, code, C):
    """The C-ABI on buffers next to pages that may not be touched, in either direction, rows at odd addresses."""
    rows, n, k, K = 3, 2, min(5, C + 1), 4
    nbytes = lib.k2amd_token_logprobs_scratch_bytes(rows, C, k, code)
    scratch = Fenced((nbytes,), np.uint8, at=at)
    rng = np.random.default_rng(C)
    if dtype == np.float32:
        x = rng.standard_normal((rows, C)).astype(np.float32)
    else:
        torch_type = torch.float16 if code == 2 else torch.bfloat16
        x = torch.from_numpy(rng.standard_normal((rows, C))).to(torch_type).view(torch.int16).numpy().view(np.uint16)
    fx = fenced(x, at)
    tokens = fenced(rng.integers(0, C, (rows, n)), at)
    mask = fenced(np.array([1, 0, 1], dtype=np.uint8), at)
    f32 = lambda *shape: Fenced(shape, np.float32, fill=np.nan, at=at)  # noqa: E731
    lp, h, tl, stats = f32(rows, n), f32(rows), f32(rows, k), f32(rows, 2)
    tt = Fenced((rows, k), np.int64, fill=-7, at=at)
    assert lib.k2amd_token_logprobs_forward(p(fx), C, p(tokens), p(mask), p(lp), p(h), p(tl), p(tt), p(stats), rows, C, n, k,
                                            1.0, code, p(scratch), nbytes, None) == 0
    assert scratch.intact()
    for f in (lp, h, stats):
        assert np.isfinite(f.a).all() and f.intact()
    assert (tt.a[0][:min(k, C)] >= 0).all() and (tt.a[1] == -1).all() and tt.intact() and tl.intact()
    grads = [fenced(np.ones((rows, n), np.float32), at), fenced(np.ones(rows, np.float32), at), fenced(np.ones((rows, k), np.float32), at)]
    dx = Fenced((rows, C), dtype, fill=77, at=at)
    assert lib.k2amd_token_logprobs_backward(p(fx), C, p(tokens), p(mask), p(stats), p(h), p(tt), *(p(g) for g in grads), p(dx),
                                             rows, C, n, k, 1.0, code, None) == 0
    assert dx.intact() and (dx.a[1] == 0).all() and not (dx.a[0] == 77).any()
    entries = rng.integers(-1, C, (rows, K))
    entries[0, 0] = C - 1
    ft, fa = fenced(entries, at), fenced(np.log(np.full((rows, K), 0.2, np.float32)), at)
    for rest in (0, 1):
        losses, records = f32(rows), f32(rows, 4)
        dbytes = lib.k2amd_distillation_scratch_bytes(rows, C, code)
        dscratch = Fenced((dbytes,), np.uint8, at=at)
        dx = Fenced((rows, C), dtype, fill=77, at=at)
        up = fenced(np.ones(rows, np.float32), at)
        assert lib.k2amd_distillation_forward(p(fx), C, p(fa), p(ft), p(mask), p(losses), p(records), rows, C, K, rest, 1.0, code,
                                              p(dscratch), dbytes, None) == 0
        assert lib.k2amd_distillation_backward(p(fx), C, p(fa), p(ft), p(records), p(up), 1, None, 1.0, p(dx), rows, C, K, rest,
                                               1.0, code, None) == 0
        assert np.isfinite(losses.a).all() and losses.intact() and dscratch.intact() and records.intact() and dx.intact()
        assert (dx.a[1] == 0).all() and not (dx.a[0] == 77).any()
        nbytes = lib.k2amd_distillation_sum_scratch_bytes(1, rows)
        scratch, out, inv = Fenced((nbytes,), np.uint8, at=at), f32(1), f32(1)
        assert lib.k2amd_distillation_sum(p(losses), p(mask), p(out), p(inv), 1, rows, 1, 1.0, p(scratch), nbytes, None) == 0
        np.testing.assert_allclose(out.a[0], losses.a.sum() / 2, rtol=1e-6, atol=1e-7)
        assert inv.a[0] == 0.5 and out.intact() and inv.intact() and scratch.intact()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 40, 700, 2300])
def test_rows_of_nothing_get_no_gradient(host, C, dtype):
    """A row of nothing but -inf: log-probs that no logit moves, whichever of them are asked for."""
    import k2_amd as k2
    x = orc.logits_case(C, 3, C, dtype, CPU)
    x[1] = NEG
    x.requires_grad_()
    got = k2.get_token_logprobs(x, torch.tensor([[0, C - 1]] * 3), num_top=2, return_entropy=True)
    assert got.logprobs[1].eq(NEG).all() and got.entropy[1] == 0 and got.top_logprobs[1].eq(NEG).all()
    ups = [torch.full_like(u, 3.0) for u in (got.logprobs, got.entropy, got.top_logprobs)]
    ups[0][1, 0] = float("inf")  # what a loss of exp(-logprob) would send back
    (grad,) = torch.autograd.grad([got.logprobs, got.entropy, got.top_logprobs], x, ups)
    assert grad[1].eq(0).all()
    assert C == 1 or (grad[0].ne(0).any() and grad[2].ne(0).any())


@pytest.mark.parametrize("temperature", [1e-50, 1e-40, 4e-39, 1e39])
def test_temperatures_out_of_range(host, temperature):
    """log2 e / temperature has to be a float32 number."""
    import k2_amd as k2
    x = torch.randn(3, 9)
    with pytest.raises(Exception, match="invalid argument"):
        k2.get_token_logprobs(x, torch.zeros(3, dtype=torch.int64), temperature=temperature)
    with pytest.raises(Exception, match="invalid argument"):
        k2.distillation_loss(x, torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64), temperature=temperature)
    got = k2.get_token_logprobs(x, temperature=5e-39, num_top=1, return_entropy=True)
    assert got.top_logprobs.eq(0).all() and got.entropy.eq(0).all()


def test_entry_points_refuse_before_launching():
    """On the library itself: wrong arguments come back as codes; pointers are never looked at."""
    import ctypes
    from k2_amd import capi
    lib = capi.lib()
    one = ctypes.c_void_p(1)

    def forward(rows=1, C=8, n=0, k=0, tau=1.0, dtype=0, x=one, stride=8, tokens=one, out=one, scratch=None, size=0):
        return lib.k2amd_token_logprobs_forward(x, stride, tokens, None, out, None, out, out, None, rows, C, n, k, tau, dtype,
                                                scratch, size, None)

    assert forward(rows=0) == 0
    assert [forward(rows=-1), forward(C=0), forward(n=-1), forward(k=-1), forward(dtype=1), forward(dtype=9), forward(x=None),
            forward(stride=-8), forward(n=1, tokens=None), forward(n=1, out=None), forward(k=1, out=None)] == [1] * 11
    assert [forward(tau=t) for t in (0.0, -1.0, float("inf"), float("nan"))] == [1] * 4
    assert [forward(n=65), forward(k=65), forward(rows=1 << 31), forward(C=(1 << 20) + 1)] == [2] * 4
    # rows longer than a workgroup holds need scratch
    need = lib.k2amd_token_logprobs_scratch_bytes(3000, 40000, 5, 3)
    assert need == 3000 * 2 * (16 + 5 * 8) and lib.k2amd_token_logprobs_scratch_bytes(3000, 32000, 5, 3) == 0
    ok = ctypes.c_void_p(16)
    for scratch, size in ((None, 0), (ok, need - 1), (one, need)):
        assert forward(rows=3000, C=40000, k=5, dtype=3, scratch=scratch, size=size) == 3

    def distill(rows=1, C=8, K=1, tau=1.0, dtype=3, x=one, a=one, out=one):
        return lib.k2amd_distillation_forward(x, 8, a, a, None, out, None, rows, C, K, 0, tau, dtype, None, 0, None)

    assert distill(rows=0) == 0 and distill(K=257) == 2 and distill(rows=1 << 31) == 2
    assert distill(C=200000) == 3 and lib.k2amd_distillation_scratch_bytes(3000, 100000, 2) == 3000 * 2 * 8
    assert [distill(rows=-1), distill(C=0), distill(K=-1), distill(tau=0.0), distill(dtype=1), distill(x=None), distill(a=None),
            distill(out=None)] == [1] * 8
    back = lambda per, g=one: lib.k2amd_distillation_backward(one, 8, one, one, one, g, per, None, 1.0, one, 1, 8, 1, 0, 1.0, 0, None)  # noqa: E731
    assert back(0) == 1 and back(1, None) == 1
    assert lib.k2amd_token_logprobs_backward(one, 8, None, None, one, None, None, one, None, None, one, 1, 8, 1, 0, 1.0, 0, None) == 1
    assert lib.k2amd_token_logprobs_backward(one, 8, one, None, one, None, None, None, one, None, one, 1, 8, 1, 0, 1.0, 0, None) == 1
    assert lib.k2amd_distillation_sum(one, None, one, None, 1, 20000, 0, 1.0, ok, 159, None) == 3
    assert lib.k2amd_distillation_sum(one, None, one, None, 1, 20000, 0, 1.0, one, 160, None) == 3
    assert lib.k2amd_distillation_sum(one, None, one, None, 1, -1, 0, 1.0, one, 8, None) == 1
    assert lib.k2amd_distillation_sum(None, None, None, None, 0, 0, 0, 1.0, None, 0, None) == 0
    assert lib.k2amd_distillation_sum_scratch_bytes(2, 10) == 0 and lib.k2amd_distillation_sum_scratch_bytes(2, 20000) == 2 * 160
    assert lib.k2amd_rnnt_pruned_mask(None, None, None, 0, 3, 3, None) == 0
    assert lib.k2amd_rnnt_pruned_mask(None, None, None, 1, 3, 3, None) == 1
    assert lib.k2amd_rnnt_pruned_mask(one, one, one, 1 << 20, 1 << 11, 1, None) == 2


def test_python_refusals(host):
    import k2_amd as k2
    x = torch.randn(4, 9)
    tokens, a, t = torch.zeros(4, dtype=torch.int64), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    for bad in (dict(temperature=0.0), dict(temperature=float("nan")), dict(num_top=65), dict(num_top=-1),
                dict(tokens=tokens[:3]), dict(tokens=torch.zeros(4, 65, dtype=torch.int64)), dict(tokens=tokens.int()),
                dict(tokens=torch.zeros(4, 0, dtype=torch.int64)), dict(mask=torch.ones(4)), dict(mask=torch.ones(3, dtype=torch.bool))):
        with pytest.raises(AssertionError):
            k2.get_token_logprobs(x, **bad)
    for bad in (dict(temperature=-1.0), dict(mask=torch.ones(4, 9, dtype=torch.bool)), dict(top_tokens=t[:, :1]),
                dict(top_tokens=t.int()), dict(top_logprobs=a.long()), dict(top_logprobs=a.clone().requires_grad_()),
                dict(top_logprobs=a[:3], top_tokens=t[:3]), dict(top_logprobs=a[:, :0], top_tokens=t[:, :0]),
                dict(top_logprobs=torch.zeros(4, 257), top_tokens=torch.zeros(4, 257, dtype=torch.int64))):
        with pytest.raises(AssertionError):
            k2.distillation_loss(x, **{**dict(top_logprobs=a, top_tokens=t), **bad})
    for bad in (dict(rest="drop"), dict(reduction="max"), dict(reduction=None)):
        with pytest.raises(ValueError):
            k2.distillation_loss(x, a, t, **bad)
    with pytest.raises(AssertionError):
        k2.rnnt_distillation_loss_pruned(x, a, t, torch.zeros(1, 4, 1, dtype=torch.int64))
    with pytest.raises(AssertionError):
        k2.get_pruned_mask(torch.zeros(2, 3, 4, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        k2.get_token_logprobs(x.double())
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        k2.distillation_loss(x.double(), a, t)


def test_host_tensors_are_refused():
    import k2_amd as k2
    x = torch.randn(4, 9)
    with pytest.raises(RuntimeError, match="no CPU path"):
        k2.get_token_logprobs(x)
    with pytest.raises(RuntimeError, match="no CPU path"):
        k2.distillation_loss(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        k2.get_pruned_mask(torch.zeros(2, 3, 4, dtype=torch.int64), torch.zeros(2, 4, dtype=torch.int64))


def test_host_layers_refuse_tensors_that_do_not_fit(hosts):  # noqa: F811
    """The C++ and the ctypes host, called directly: a tensor of another shape or type never reaches a kernel."""
    native, capi = hosts
    x, tokens = torch.randn(4, 9), torch.zeros(4, dtype=torch.int64)
    stats, a, t = torch.zeros(4, 2), torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int64)
    for host_layer in (native._ext, capi):
        for call in (lambda: host_layer.token_logprobs_forward(x, tokens[:3], None, 1.0, 0, False, False),
                     lambda: host_layer.token_logprobs_forward(x, tokens, torch.ones(4), 1.0, 0, False, False),
                     lambda: host_layer.token_logprobs_forward(x, tokens, None, 1.0, 65, False, False),
                     lambda: host_layer.token_logprobs_forward(x, tokens, None, 1.0, -1, False, False),
                     lambda: host_layer.token_logprobs_forward(x, tokens, None, 0.0, 0, False, False),
                     lambda: host_layer.token_logprobs_backward(x, tokens, None, stats[:3], None, None, None, None, None, 1.0),
                     lambda: host_layer.token_logprobs_backward(x, tokens, None, stats, None, None, torch.zeros(3), None, None, 1.0),
                     lambda: host_layer.token_logprobs_backward(x, None, None, stats, None, None, torch.zeros(4), None, None, 1.0),
                     lambda: host_layer.distillation_forward(x, a, t[:3], None, 1.0, False, False),
                     lambda: host_layer.distillation_forward(x, a.half(), t, None, 1.0, False, False),
                     lambda: host_layer.distillation_backward(x, a, t, torch.zeros(4, 3), torch.zeros(4), None, 1.0, 1.0, False),
                     lambda: host_layer.distillation_backward(x, a, t, torch.zeros(4, 4), torch.zeros(3), None, 1.0, 1.0, False),
                     lambda: host_layer.distillation_sum(torch.zeros(7), None, 2, False, 1.0),
                     lambda: host_layer.pruned_mask(torch.zeros(2, 3, 4, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int64)),
                     lambda: host_layer.pruned_mask(torch.zeros(2, 3, 4, dtype=torch.int64), torch.zeros(2, 3, dtype=torch.int64))):
            with pytest.raises(RuntimeError):
                call()


def test_half_conversion_of_the_host_build_is_the_hardware_rounding():
    """tests/cpu_build/hip/hip_runtime.h rounds to half precision as IEEE does: every half there and back, and midpoints."""
    import subprocess
    import os
    src = os.path.join(ck.OUT, "half.cc")
    os.makedirs(ck.OUT, exist_ok=True)
    with open(src, "w") as f:
        f.write('#include "hip/hip_runtime.h"\nextern "C" unsigned short to_half(float f) { return hip_threads_to_half(f); }\n')
    out = os.path.join(ck.OUT, "libhalf.so")
    subprocess.run(["g++", *ck.FLAGS, "-shared", "-x", "c++", src, "-o", out], check=True)
    import ctypes
    fn = ctypes.CDLL(out).to_half
    fn.argtypes, fn.restype = [ctypes.c_float], ctypes.c_ushort
    halves = np.arange(0, 0x7c00, 17, dtype=np.uint16).view(np.float16).astype(np.float32)
    mid = (halves[:-1] + halves[1:]) / 2
    values = np.concatenate([halves, mid, np.nextafter(mid, np.float32(0)), [65519.0, 65520.0, 1e9, 3e-8, 2.9e-8, 1e-9, np.inf]])
    for v in np.concatenate([values, -values]).astype(np.float32):
        with np.errstate(over="ignore"):
            assert fn(float(v)) == int(np.float16(v).view(np.uint16)), v
