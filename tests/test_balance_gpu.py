"""Balance loss of the router on the GPU against its definition in 64 bits.

Tolerances: p is a quotient of fp32 sums of at most E exponentials, each off by a few ulp: (E / 32 + 5
shuffle steps + 16) 2^-23 relative covers the sum, the fast exponentials (2 ulp and 2^-24 of their
argument, |l - max| <= 40 here: 2^-18 in the worst term, which then weighs exp(-40)) and the
divisions, so 2^-18 of the sum of the absolute terms bounds a loss and each gradient's terms.
Gradients are also rounded once to the logits' type."""

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda:0"
SOFTMAX, SIGMOID = 0, 1


def _nat():
    from distributedmoe_b200 import _native as N
    return N


def _reference(l, idx, mode, seq_end, mask, ga, gz):
    """(balance, z, counts, gradient, sum of absolute gradient terms) by the definition."""
    T, E = l.shape
    k = idx.shape[1]
    l = l.detach().double()
    ends = [T] if seq_end is None else seq_end.tolist()
    keep = torch.ones(T, dtype=torch.bool, device=l.device) if mask is None else mask.bool()
    seq = torch.full((T,), -1, device=l.device)
    a = 0
    for s, b in enumerate(ends):
        seq[a:b] = s
        a = max(a, b)
    keep = keep & (seq >= 0)
    S = len(ends)
    counts = torch.zeros(S, E, dtype=torch.int64, device=l.device)
    for s in range(S):
        sel = idx[keep & (seq == s)].flatten()
        sel = sel[(sel >= 0) & (sel < E)]
        counts[s] = torch.bincount(sel, minlength=E)
    n = torch.stack([(keep & (seq == s)).sum() for s in range(S)]) if S else torch.zeros(0, device=l.device)
    full, total = int((n > 0).sum()), int(n.sum())
    some = keep & (l.amax(1) > float("-inf"))
    rows = l[some]
    soft = torch.softmax(rows, 1)
    lse = torch.logsumexp(rows, 1)
    if mode == SOFTMAX:
        p, slope = soft, torch.ones_like(soft)
    else:
        p, slope = torch.softmax(torch.nn.functional.logsigmoid(rows), 1), torch.sigmoid(-rows)
    c = counts.double()[seq[some]]
    coef = (E / (k * n.double() ** 2 * max(full, 1)))[seq[some]]
    dot = (c * p).sum(1)
    balance = float((coef * dot).sum())
    z = float((lse ** 2).sum() / max(total, 1))
    grad, size = torch.zeros_like(l), torch.zeros_like(l)
    grad[some] = ga * coef[:, None] * p * slope * (c - dot[:, None]) + gz * 2 / max(total, 1) * lse[:, None] * soft
    size[some] = abs(ga) * coef[:, None] * p * slope * (c + dot[:, None]) + abs(gz) * 2 / max(total, 1) * lse.abs()[:, None] * soft
    return balance, z, counts, grad, size


def _check(l, idx, mode, seq_end=None, mask=None, ga=0.7, gz=0.3):
    N = _nat()
    balance, z, counts = N.balance_loss(l, idx, mode=mode, seq_end=seq_end, mask=mask)
    up = [torch.tensor(v, device=DEV) for v in (ga, gz)]
    grad, = torch.autograd.grad([balance, z], [l], up)
    rb, rz, rc, rg, size = _reference(l, idx, mode, seq_end, mask, ga, gz)
    balance, z = balance.detach(), z.detach()
    assert counts.dtype == torch.int32 and torch.equal(counts.long(), rc)
    assert abs(float(balance) - rb) <= 2.0 ** -18 * abs(rb)
    assert abs(float(z) - rz) <= 2.0 ** -18 * (abs(rz) + 1)  # + 1: lse near 0 is a difference
    eps = torch.finfo(l.dtype).eps
    smallest = torch.finfo(l.dtype).tiny
    off = (grad.double() - rg).abs() - (2.0 ** -18 * size + eps / 2 * rg.abs() + smallest)
    assert off.max().item() <= 0 if off.numel() else True
    N.check_device_status(torch.device(DEV))
    return balance, z, counts, grad


def _case(T, E, k, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    l = (2.0 * torch.randn(T, E, generator=g, device=DEV)).to(dtype)
    idx = torch.topk(l.float(), k, dim=1).indices.contiguous() if T else torch.empty(0, k, dtype=torch.int64, device=DEV)
    return l.requires_grad_(True), idx


@gpu
@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 5, 3), (33, 8, 1), (1000, 16, 4), (257, 33, 2), (515, 64, 8),
                                   (300, 100, 6), (1031, 256, 8), (65, 511, 5), (40, 1024, 16), (9000, 8, 2)])
def test_one_sequence(T, E, k, dtype, mode):
    _check(*_case(T, E, k, dtype, T + E), mode)


@gpu
@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("T,E,k,ends", [
    (100, 8, 2, [0, 0, 1, 50, 50, 99]),           # empty sequences, one token, one token behind the last
    (700, 100, 4, [13, 14, 400, 700, 700]),
    (2000, 256, 8, list(range(7, 2000, 61))),
    (5, 8, 2, [0, 0]),                              # every token behind the last sequence
    (64, 32, 2, list(range(1, 65))),                # a sequence a token
])
@pytest.mark.parametrize("masked", [0.0, 0.5, 1.0])
def test_sequences_and_masks(T, E, k, ends, mode, masked):
    l, idx = _case(T, E, k, torch.float32, T)
    seq_end = torch.tensor(ends, dtype=torch.int32, device=DEV)
    mask = None
    if masked:
        mask = torch.rand(T, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) >= masked
        with torch.no_grad():  # what stands in masked places is not read
            l[~mask] = float("nan")
            l[~mask, 0] = float("inf")
        idx[~mask] = 2**40
    _, _, _, grad = _check(l, idx, mode, seq_end, mask)
    if masked:
        assert int(grad[~mask].count_nonzero()) == 0


@gpu
def test_no_tokens():
    N = _nat()
    l, idx = _case(0, 8, 2, torch.float32, 1)
    balance, z, counts = N.balance_loss(l, idx)
    assert float(balance.detach()) == 0 and float(z.detach()) == 0 and counts.tolist() == [[0] * 8]
    assert torch.autograd.grad(balance, l)[0].shape == (0, 8)
    l, idx = _case(4, 8, 2, torch.float32, 1)
    balance, z, counts = N.balance_loss(l, idx, seq_end=torch.empty(0, dtype=torch.int32, device=DEV))
    assert float(balance) == 0 and float(z) == 0 and counts.shape == (0, 8)
    assert int(torch.autograd.grad(balance + z, l)[0].count_nonzero()) == 0


@gpu
@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("E", [8, 100, 256])
def test_extreme_logits(E, mode):
    """Experts masked by -inf or by the type's lowest value, rows with nothing left, rows far from
    zero whose sigmoids all round to 0 or 1."""
    l, idx = _case(64, E, 2, torch.float32, E)
    with torch.no_grad():
        l[0::8, :3] = float("-inf")
        l[1::8] = float("-inf")
        l[2::8, 1:] = torch.finfo(torch.float32).min
        l[3::8] -= 200.0
        l[4::8] += 200.0
        l[5::8, 2] = 90.0
    _check(l, idx, mode, ga=0.7, gz=0.0)
    with torch.no_grad():
        l[2::8, 1:] = -300.0
    _check(l, idx, mode)


@gpu
@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
def test_nan_and_inf_are_not_hidden(mode):
    N = _nat()
    l, idx = _case(20, 64, 2, torch.float32, 1)
    with torch.no_grad():
        l[7, 9] = float("nan")
    balance, z, _ = N.balance_loss(l, idx, mode=mode)
    assert balance.isnan() and z.isnan()
    grad, = torch.autograd.grad(balance, l)
    assert bool(grad[7].isnan().all()) and bool(grad[:7].isfinite().all()) and bool(grad[8:].isfinite().all())


@gpu
def test_dropped_and_repeated_selections():
    l, idx = _case(50, 8, 3, torch.float32, 2)
    idx[::3, 1] = -1
    idx[1::3, 2] = 8
    idx[2::3] = 5
    _check(l, idx, SOFTMAX)


@gpu
@pytest.mark.parametrize("mode", [SOFTMAX, SIGMOID])
def test_gradient_against_differences(mode):
    """Central differences of the losses in 64 bits (their counts held), at a step whose third-order
    term is below 1e-6 of the gradient's largest."""
    l, idx = _case(12, 9, 2, torch.float32, 4)
    seq_end = torch.tensor([5, 12], dtype=torch.int32, device=DEV)
    _, _, _, grad = _check(l, idx, mode, seq_end)
    step, base = 1e-4, l.detach().double()
    num = torch.zeros_like(base)
    for i in range(12):
        for j in range(9):
            v = []
            for sign in (1, -1):
                x = base.clone()
                x[i, j] += sign * step
                b, z, *_ = _reference(x, idx, mode, seq_end, None, 0.0, 0.0)
                v.append(0.7 * b + 0.3 * z)
            num[i, j] = (v[0] - v[1]) / (2 * step)
    assert ((grad.double() - num).abs().max() / num.abs().max()).item() <= 1e-5


@gpu
def test_one_loss_alone():
    """A loss that is not used costs no gradient and needs none."""
    N = _nat()
    l, idx = _case(100, 64, 4, torch.float32, 4)
    for which, (ga, gz) in ((0, (1.0, 0.0)), (1, (0.0, 1.0))):
        out = N.balance_loss(l, idx, mode=SIGMOID)
        grad, = torch.autograd.grad(out[which], l)
        rg, size = _reference(l, idx, SIGMOID, None, None, ga, gz)[3:]
        assert bool(((grad.double() - rg).abs() <= 2.0 ** -18 * size + 2.0 ** -24 * rg.abs() + 1e-37).all())
    assert not out[2].requires_grad


@gpu
def test_after_the_router():
    """Router, its balance loss and a training step's gradient, as they are used together."""
    N = _nat()
    g = torch.Generator(device=DEV).manual_seed(6)
    T, d, E, k = 200, 256, 16, 4
    x = torch.randn(T, d, generator=g, device=DEV).to(torch.bfloat16)
    w_r = (0.05 * torch.randn(E, d, generator=g, device=DEV)).to(torch.bfloat16)
    idx, _, logits = N.router(x, w_r, k, want_logits=True)
    plan = N.route_plan(idx, None, E, want_weight=False)
    l = (x.float() @ w_r.float().T).requires_grad_(True)
    balance, z, counts = N.balance_loss(l, idx)
    assert torch.equal(counts[0], plan["counts"])
    (0.01 * balance + 0.001 * z).backward()
    rg, size = _reference(l, idx, SOFTMAX, None, None, 0.01, 0.001)[3:]
    assert bool(((l.grad.double() - rg).abs() <= 2.0 ** -18 * size + 2.0 ** -23 * rg.abs()).all())
    assert N.balance_loss(logits, idx)[0].requires_grad is False


@gpu
def test_captured_forward_and_backward():
    """Forward and backward in one graph, replayed on new logits."""
    N = _nat()
    l, idx = _case(500, 64, 4, torch.float32, 8)
    up = torch.ones((), device=DEV)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(N.balance_loss(l, idx)[0], l, up)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        balance, z, counts = N.balance_loss(l, idx)
        grad, = torch.autograd.grad(balance, l, up)
    for seed in (1, 2):
        with torch.no_grad():
            l.copy_(_case(500, 64, 4, torch.float32, seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        rb, _, rc, rg, size = _reference(l, idx, SOFTMAX, None, None, 1.0, 0.0)
        assert abs(float(balance) - rb) <= 2.0 ** -18 * rb and torch.equal(counts.long(), rc)
        assert bool(((grad.double() - rg).abs() <= 2.0 ** -18 * size + 2.0 ** -24 * rg.abs() + 1e-37).all())


@gpu
def test_same_bits_every_time():
    N = _nat()
    l, idx = _case(20000, 64, 4, torch.float32, 8)
    seq_end = torch.arange(100, 20001, 199, dtype=torch.int32, device=DEV)
    first = N.balance_loss(l, idx, seq_end=seq_end)
    for _ in range(5):
        for a, b in zip(first, N.balance_loss(l, idx, seq_end=seq_end)):
            assert torch.equal(a, b)


@gpu
def test_bad_sequences_are_reported():
    N = _nat()
    l, idx = _case(20, 8, 2, torch.float32, 1)
    for ends in ([5, 3, 20], [5, 21], [-1, 20]):
        N.balance_loss(l, idx, seq_end=torch.tensor(ends, dtype=torch.int32, device=DEV))
        with pytest.raises(N.DMoEError, match="segment"):
            N.check_device_status(torch.device(DEV))


@gpu
def test_wrapper_refusals():
    N = _nat()
    l, idx = _case(20, 8, 2, torch.float32, 1)
    i32 = dict(dtype=torch.int32, device=DEV)
    for call in (lambda: N.balance_loss(l.double(), idx), lambda: N.balance_loss(l, idx.int()),
                 lambda: N.balance_loss(l, idx[:10]), lambda: N.balance_loss(l[0], idx), lambda: N.balance_loss(l.T, idx),
                 lambda: N.balance_loss(l, idx, mode=4), lambda: N.balance_loss(l, idx, seq_end=torch.tensor([20], device=DEV)),
                 lambda: N.balance_loss(l, idx, mask=torch.ones(19, dtype=torch.bool, device=DEV)),
                 lambda: N.balance_loss(l, idx, mask=torch.ones(20, device=DEV)),
                 lambda: N.balance_loss(l, idx, seq_end=torch.ones(1, dtype=torch.int32)),
                 lambda: N.balance_loss(torch.zeros(4, 1025, device=DEV), idx[:4]),
                 lambda: N.balance_loss(l, torch.zeros(20, 9, dtype=torch.int64, device=DEV))):
        with pytest.raises(N.DMoEError):
            call()
    assert N.balance_loss(l, idx, seq_end=torch.tensor([20], **i32))[2].shape == (1, 8)


@gpu
def test_differentiable_once():
    N = _nat()
    l, idx = _case(20, 8, 2, torch.float32, 1)
    balance, z, _ = N.balance_loss(l, idx)
    grad, = torch.autograd.grad(balance + z, l, create_graph=True)
    plain, = torch.autograd.grad(sum(N.balance_loss(l, idx)[:2]), l)
    assert torch.equal(grad.detach(), plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), l)


@gpu
def test_counts_are_the_callers():
    """Adding to the returned counts (other ranks' selections) leaves the gradient as it was."""
    N = _nat()
    l, idx = _case(50, 8, 2, torch.float32, 3)
    want, = torch.autograd.grad(N.balance_loss(l, idx)[0], l)
    balance, _, counts = N.balance_loss(l, idx)
    counts += 1000
    assert torch.equal(torch.autograd.grad(balance, l)[0], want)


@gpu
@pytest.mark.parametrize("masked", [False, True])
def test_as_many_tokens_as_there_may_be(masked):
    """T * k = 2^31 - 2: the grid, the last CTA's steps and every index at the limit that is stated.  With
    one expert the balance is 1 and z the mean of the squared logits."""
    N = _nat()
    T = 2**31 - 2
    g = torch.Generator(device=DEV).manual_seed(3)
    idx = torch.zeros(T, 1, dtype=torch.int64, device=DEV)
    l = torch.empty(T, 1, dtype=torch.bfloat16, device=DEV).normal_(generator=g).requires_grad_(True)
    mask = None
    if masked:
        mask = torch.ones(T, dtype=torch.uint8, device=DEV)
        mask[::3] = 0
    balance, z, counts = N.balance_loss(l, idx, mask=mask)
    grad, = torch.autograd.grad(z, l)
    kept, total = 0, 0.0
    for a in range(0, T, 2**28):
        b = min(T, a + 2**28)
        v = l.detach()[a:b, 0].double() ** 2
        if masked:
            v *= mask[a:b]
        total += float(v.sum())
        kept += int(mask[a:b].sum()) if masked else b - a
    N.check_device_status(torch.device(DEV))
    assert counts.tolist() == [[kept]]
    assert abs(float(balance.detach()) - 1.0) <= 2.0 ** -18 and abs(float(z.detach()) - total / kept) <= 2.0 ** -18 * (total / kept + 1)
    for part in (slice(0, 1000), slice(T - 1000, T)):
        want = 2.0 / kept * l.detach()[part].double()
        if masked:
            want *= mask[part, None]
        assert bool(((grad[part].double() - want).abs() <= (2.0 ** -18 + 2.0 ** -8) * want.abs()).all())


@gpu
def test_losses_are_the_callers():
    """Each loss may be changed in place, by itself or for logging, without touching the other one or the
    gradient that its new value has."""
    N = _nat()
    l, idx = _case(50, 8, 2, torch.float32, 3)
    want_b, want_z, _ = (t.detach().clone() for t in N.balance_loss(l, idx))
    both, = torch.autograd.grad(sum(N.balance_loss(l, idx)[:2]), l)
    balance, z, _ = N.balance_loss(l, idx)
    assert balance.shape == () and z.shape == ()
    balance *= 0.5
    assert torch.equal(balance.detach(), want_b * 0.5) and torch.equal(z.detach(), want_z)
    z *= 0.25
    balance += z
    assert torch.equal(balance.detach(), want_b * 0.5 + want_z * 0.25) and torch.equal(z.detach(), want_z * 0.25)
    grad, = torch.autograd.grad(balance, l)
    up = [torch.tensor(v, device=DEV) for v in (0.5, 0.25)]
    assert torch.equal(grad, torch.autograd.grad(N.balance_loss(l, idx)[:2], l, up)[0])
    balance, z, _ = N.balance_loss(l, idx)
    balance.detach().zero_()
    assert float(balance.detach()) == 0 and torch.equal(z.detach(), want_z)
    assert torch.equal(torch.autograd.grad(balance + z, l)[0], both)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E", [(6, 5), (300, 33), (6, 128), (4000, 12)])
def test_logits_that_start_at_any_value(T, E, dtype):
    """A contiguous slice whose first value is aligned to its type and to nothing more, small and large."""
    l, idx = _case(T, E, 2, dtype, E)
    wide = torch.full((T * E + 9,), float("nan"), dtype=dtype, device=DEV)
    for at in (1, 3, 4):
        part = wide[at:at + T * E].view(T, E)
        part.copy_(l.detach())
        _check(part.detach().requires_grad_(True), idx, SIGMOID)
        wide[at:at + T * E] = float("nan")
