"""The entity-prediction operators against plain 64-bit computations (on the CPU): ``ops.embedding`` and its gradient,
``ops.topk_distill_loss`` and its gradient, ``ops.mx4_quantize`` / ``mx4_dequantize`` / ``mx4_linear``.

Tolerances.  u = 2^-24 is half a step of fp32 (relative), h = finfo(type).eps / 2 half a step of the result's type, t its
half step at zero (smallest_normal * eps / 2, where values stop being relative).  A sum of c fp32 terms is within
(c + 2) u sum|terms| of the exact one in any order; a product or a conversion adds one half step."""
import math

import pytest
import torch
import torch.utils.checkpoint

from biomedkg_amd import _lib as L
from biomedkg_amd import ops

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def check(got, want, bound):
    """|got - want| <= bound elementwise; NaN and infinities where ``want`` has them."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    bound = bound.cpu() if torch.is_tensor(bound) else torch.full_like(want, bound)
    fin = torch.isfinite(want)
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    over = (got - want).abs()[fin] - bound.expand_as(want)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, (float(over.max()), int((over > 0).sum()))


# ----------------------------------------------------------------------------- plain forms, 64 bits
def plain_embedding(w, ids, scale):
    w, ids = w.double().cpu(), ids.long().cpu()
    ok = (ids >= 0) & (ids < w.size(0))
    rows = w[ids.clamp(0, w.size(0) - 1)] if w.size(0) else w.new_zeros(ids.shape + (w.size(1),))
    return torch.where(ok[..., None], rows, torch.zeros((), dtype=torch.float64)) * scale


def plain_embedding_grad(g, ids, v, scale, pad):
    """-> the gradient and, for the bound, the sums of magnitudes and the counts"""
    g, ids = g.double().cpu().reshape(-1, g.size(-1)), ids.long().cpu().reshape(-1)
    ok = (ids >= 0) & (ids < v)
    if pad is not None:
        ok &= ids != pad
    dw, mag = torch.zeros(v, g.size(1), dtype=torch.float64), torch.zeros(v, g.size(1), dtype=torch.float64)
    cnt = torch.zeros(v, dtype=torch.float64)
    dw.index_add_(0, ids[ok], g[ok])
    mag.index_add_(0, ids[ok], g[ok].abs())
    cnt.index_add_(0, ids[ok], torch.ones(int(ok.sum()), dtype=torch.float64))
    return dw * scale, mag * abs(scale), cnt


def check_embedding(w, ids, scale, pad, g, out, dw):
    h, t = half_step(w.dtype)
    want = plain_embedding(w, ids, scale)
    check(out, want, want.abs() * (h + 2 * U) + t)
    want, mag, cnt = plain_embedding_grad(g, ids, w.size(0), scale, pad)
    check(dw, want, want.abs() * h + (cnt[:, None] + 4) * U * mag * (1 + h) + t)


def run_embedding(w, ids, scale, pad, g):
    w = w.detach().requires_grad_()
    out = ops.embedding(w, ids, scale=scale, padding_idx=pad)
    out.backward(g)
    return out, w.grad


# ----------------------------------------------------------------------------- embedding
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,d,n", [(1, 1, 1), (7, 3, 5), (5000, 768, 1021), (300, 256, 9001), (130, 8, 700), (64, 130, 1),
                                   (97, 513, 3000), (20000, 64, 12), (1000, 1100, 333), (40, 20, 20000), (3, 260, 2000)])
def test_embedding_and_gradient(dtype, v, d, n):
    gen = torch.Generator().manual_seed(v * 1000 + d + n)
    w = torch.randn(v, d, generator=gen).to(dtype).cuda()
    ids = (torch.rand(n, generator=gen).pow(3) * v).long().clamp_(max=v - 1).cuda()
    g = torch.randn(n, d, generator=gen).to(dtype).cuda()
    out, dw = run_embedding(w, ids, 1.75, None, g)
    check_embedding(w, ids, 1.75, None, g, out, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("runs", [[257], [256], [255, 2], [1, 256, 1], [1, 257, 1], [512, 512], [600, 3, 700, 1, 1, 5000],
                                  [255, 257, 255, 300], [10000]])
@pytest.mark.parametrize("shuffle", [False, True])
def test_embedding_gradient_of_long_runs(runs, shuffle):
    """run lengths on both sides of the split, runs that begin and end at every place of a window"""
    gen = torch.Generator().manual_seed(sum(runs))
    ids = torch.repeat_interleave(torch.arange(len(runs)) * 3 + 1, torch.tensor(runs))
    if shuffle:
        ids = ids[torch.randperm(ids.numel(), generator=gen)]
    v, d = 3 * len(runs) + 2, 72
    w = torch.randn(v, d, generator=gen).cuda()
    g = torch.randn(ids.numel(), d, generator=gen).cuda()
    out, dw = run_embedding(w, ids.cuda(), 0.5, None, g)
    check_embedding(w, ids, 0.5, None, g, out, dw)
    again = run_embedding(w, ids.cuda(), 0.5, None, g)[1]
    assert torch.equal(dw, again)                                         # fixed order: the same bits


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v,d,n", [(1, 5, 2048), (16, 64, 2047), (17, 1024, 1500), (5000, 768, 2048), (300, 7, 1), (40, 2000, 31),
                                   (2, 1030, 2), (9000, 1, 700), (70000, 24, 2049)])
def test_embedding_gradient_of_short_lists(v, d, n, dtype):
    """one hub takes a third of the ids; some lie outside the table"""
    gen = torch.Generator().manual_seed(v + d + n)
    w = torch.randn(v, d, generator=gen).to(dtype).cuda()
    ids = torch.randint(-1, v + 1, (n,), generator=gen)
    ids[torch.rand(n, generator=gen) < 0.34] = v // 2
    for pad in (None, v // 2):
        g = torch.randn(n, d, generator=gen).to(dtype).cuda()
        out, dw = run_embedding(w, ids.cuda(), -0.5, pad, g)
        check_embedding(w, ids, -0.5, pad, g, out, dw)
        again = run_embedding(w, ids.cuda(), -0.5, pad, g)[1]
        assert torch.equal(dw, again)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [2, 511, 512, 513, 130000, 262143, 262144, 3000000])
@pytest.mark.parametrize("n", [2048, 2049, 4096, 4097, 8192, 8193, 12288, 50001, 131072, 131073])
def test_embedding_gradient_over_many_rows(v, n):
    """one, two and three passes of the sort, tables with and without a spare bit above the last row"""
    gen = torch.Generator().manual_seed(v + n)
    ids = torch.randint(0, v, (n,), generator=gen)
    ids[:3] = torch.tensor([v - 1, 0, v - 1])
    w = torch.empty(v, 4).cuda()
    w.zero_()
    g = torch.randn(n, 4, generator=gen).cuda()
    out, dw = run_embedding(w, ids.cuda(), 1.0, None, g)
    check_embedding(w, ids, 1.0, None, g, out, dw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("id_type", [torch.int64, torch.int32])
def test_embedding_padding_and_outside_ids(dtype, id_type):
    v, d, n = 50, 96, 9500
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(-4, v + 4, (n,), generator=gen).to(id_type)
    ids[::5] = 49
    ids[1] = torch.iinfo(id_type).max
    ids[2] = torch.iinfo(id_type).min
    w = torch.randn(v, d, generator=gen).to(dtype).cuda()
    g = torch.randn(n, d, generator=gen).to(dtype).cuda()
    for m in (n, 700):                                                    # both sorts
        out, dw = run_embedding(w, ids[:m].cuda(), -2.0, -1, g[:m])
        check_embedding(w, ids[:m], -2.0, 49, g[:m], out, dw)
        assert float(dw[49].abs().max()) == 0.0
    none = torch.full((300,), -1, dtype=id_type).cuda()                   # nothing usable: a zero gradient
    out, dw = run_embedding(w, none, 1.0, None, g[:300])
    assert float(out.abs().max()) == 0.0 and float(dw.abs().max()) == 0.0


@pytest.mark.gpu
def test_embedding_shapes_strides_and_empty():
    gen = torch.Generator().manual_seed(4)
    big = torch.randn(40, 131, generator=gen).cuda()
    w = big[::2, 3:68]                                                     # row stride 262, start 12 bytes off
    ids = torch.randint(0, 20, (6, 5), generator=gen).cuda().t()           # not contiguous
    w2 = w.detach().requires_grad_()
    out = ops.embedding(w2, ids, scale=3.0)
    assert out.shape == (5, 6, 65)
    out.sum().backward()                                                   # an expanded upstream gradient
    check_embedding(w, ids, 3.0, None, torch.ones(5, 6, 65), out, w2.grad)
    row = torch.randn(1, 64, generator=gen).cuda().requires_grad_()        # a broadcast table: the gradient sums over it
    ops.embedding(row.expand(7, 64), ids[:, 0].contiguous() % 7).sum().backward()
    assert torch.equal(row.grad, torch.full((1, 64), 5.0, device="cuda"))
    wt = torch.randn(64, 30, generator=gen).cuda().t()                     # columns not next to each other
    assert torch.equal(ops.embedding(wt, torch.tensor(3).cuda()), wt[3])
    for shape in ((0,), (3, 0)):
        e = torch.empty(shape, dtype=torch.int64, device="cuda")
        w3 = torch.ones(4, 8, device="cuda", requires_grad=True)
        out = ops.embedding(w3, e)
        assert out.shape == shape + (8,)
        out.sum().backward()
        assert float(w3.grad.abs().max()) == 0.0
    out = ops.embedding(torch.empty(0, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert out.shape == (3, 8) and float(out.abs().max()) == 0.0


@pytest.mark.gpu
def test_embedding_gradient_against_differences():
    gen = torch.Generator().manual_seed(5)
    w = torch.randn(6, 4, generator=gen).cuda()
    ids = torch.tensor([1, 4, 1, 0, 5, 1, -1]).cuda()
    g = torch.randn(7, 4, generator=gen).cuda()
    _, dw = run_embedding(w, ids, 1.5, 5, g)
    for (r, c) in ((1, 2), (4, 0), (3, 3)):
        d = torch.zeros(6, 4, dtype=torch.float64)
        d[r, c] = 0.25
        up = (plain_embedding(w.cpu().double() + d, ids, 1.5) * g.cpu().double()).sum()
        dn = (plain_embedding(w.cpu().double() - d, ids, 1.5) * g.cpu().double()).sum()
        assert abs(float(dw[r, c]) - float((up - dn) / 0.5)) <= 8 * U * 1.5 * float(g.abs().sum())   # (linear: exact differences)


# ----------------------------------------------------------------------------- distillation
def plain_distill(x, ids, t, temp):
    """per-row losses, gradients of each row's own loss, and (p, q, range of exponents) for the bounds"""
    x, ids, t = x.double().cpu(), ids.long().cpu(), t.double().cpu()
    rows, v = x.shape
    loss, grad = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, v, dtype=torch.float64)
    pq = torch.zeros(rows, v, dtype=torch.float64)
    span = 1.0
    for r in range(rows):
        use = (ids[r] >= 0) & (ids[r] < v) & ~(t[r] == -math.inf)
        if not bool(use.any()) or bool((x[r] == -math.inf).all()):
            continue
        z = x[r] / temp
        lp = torch.log_softmax(z, 0)
        lq = torch.log_softmax(t[r][use] / temp, 0)
        q = lq.exp()
        at = ids[r][use]
        term = q * (lq - lp[at])
        loss[r] = temp * temp * torch.where(q == 0, torch.zeros_like(term), term).sum()
        p = lp.exp()
        grad[r] = temp * p
        grad[r].index_add_(0, at, -temp * q)
        pq[r] = p
        pq[r].index_add_(0, at, q)
        for a in (z, t[r][use] / temp):
            a = a[torch.isfinite(a)]
            if a.numel():
                span = max(span, float(a.max() - a.min()))
    return loss, grad, pq, span


def distill_bounds(x, k, temp, loss, grad, pq, span):
    """The exponents' arguments carry 3 u each relative, so an exponential 3 u span + 2 u; the row's sum adds one half step per
    term of a thread's chain (V / 256 at most) and of the joins; ln of a sum has its relative error as an absolute one."""
    d = U * (3 * span + x.size(1) / 256 + 2 * k + 32)
    h, t = half_step(x.dtype)
    # a row's loss: sum_j q_j (ln q_j - ln p_j), |ln| <= span + ln V
    loss_b = temp * temp * d * (4 + 2 * span + 2 * math.log(x.size(1) + 1))
    grad_b = temp * 2 * d * pq
    return loss_b, lambda scale: grad.abs() * scale * (h + 4 * U) + grad_b * scale * (1 + h) + t


def make_distill(rows, v, k, dtype, seed, t_type=torch.float32, id_type=torch.int64):
    gen = torch.Generator().manual_seed(seed)
    x = (3 * torch.randn(rows, v, generator=gen)).to(dtype)
    ids = torch.stack([torch.randperm(v, generator=gen)[:k] for _ in range(rows)])
    t = (2 * torch.randn(rows, k, generator=gen)).to(t_type)
    return x.cuda(), ids.to(id_type).cuda(), t.cuda()


def check_distill(x, ids, t, temp):
    loss, grad, pq, span = plain_distill(x, ids, t, temp)
    lb, gb = distill_bounds(x, ids.size(1), temp, loss, grad, pq, span)
    rows = x.size(0)
    g = torch.linspace(0.5, 2.0, rows)
    for red in ("none", "sum", "batchmean"):
        xx = x.detach().requires_grad_()
        got = ops.topk_distill_loss(xx, ids, t, temp, reduction=red)
        plain = ops.topk_distill_loss(x, ids, t, temp, reduction=red)
        assert torch.equal(torch.nan_to_num(got.detach(), nan=7.0), torch.nan_to_num(plain, nan=7.0))
        if red == "none":
            check(got, loss, lb)
            got.backward(g.cuda())
            check(xx.grad, grad * g[:, None], gb(g[:, None].double()))
        else:
            f = 1.0 if red == "sum" else 1.0 / rows
            check(got, loss.sum() * f, rows * lb * f + (rows + 2) * U * f * float(loss.abs().nan_to_num(0, 0, 0).sum()))
            (got * 0.75).backward()
            check(xx.grad, grad * (0.75 * f), gb(0.75 * f))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v,k,temp", [(1, 1, 1, 1.0), (3, 2, 2, 0.5), (16, 5000, 10, 2.0), (5, 32771, 64, 1.0),
                                           (130, 700, 33, 4.0), (2, 40000, 1024, 1.5), (1, 40001, 1, 1.0), (2100, 37, 5, 3.0)])
def test_distill_and_gradient(dtype, rows, v, k, temp):
    check_distill(*make_distill(rows, v, k, dtype, rows + v + k), temp)


@pytest.mark.gpu
@pytest.mark.parametrize("t_type", TYPES)
@pytest.mark.parametrize("id_type", [torch.int64, torch.int32])
def test_distill_padding_masks_and_empty_rows(t_type, id_type):
    x, ids, t = make_distill(9, 333, 6, torch.float32, 11, t_type, id_type)
    ids[0] = -1                                              # no teacher
    ids[1, 2:] = -1
    ids[2, 0], ids[2, 1] = 333, torch.iinfo(id_type).max     # outside the columns
    t[3] = -math.inf                                         # the teacher masked everything
    t[4, ::2] = -math.inf
    x[5] = -math.inf                                         # the student masked everything
    keep = torch.zeros(333, dtype=torch.bool)
    keep[ids[6].long().cpu()] = True
    x[6, ~keep.cuda()] = -math.inf                           # only the teacher's columns are left
    x[7, :300] = torch.finfo(torch.float32).min              # a mask of the type's lowest value
    ids[7] = torch.arange(300, 306)
    check_distill(x, ids, t, 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_nonfinite_stays_in_its_row(dtype):
    x, ids, t = make_distill(6, 500, 4, dtype, 12)
    x[0, 7] = math.nan
    x[1, 9] = math.inf
    x[2, ids[2, 1]] = -math.inf                              # a usable entry the student gives no mass: loss inf
    t[3, 0] = math.nan
    x[4, 3], ids[4] = math.nan, -1                           # left out whatever its logits are
    xx = x.detach().requires_grad_()
    out = ops.topk_distill_loss(xx, ids, t, 1.0, reduction="none")
    out.sum().backward()
    assert torch.isnan(out[0]) and torch.isnan(out[1]) and out[2] == math.inf and torch.isnan(out[3])
    assert out[4] == 0 and float(xx.grad[4].abs().max()) == 0
    assert bool(torch.isnan(xx.grad[0]).all()) and bool(torch.isnan(xx.grad[3, ids[3].unique()]).all())
    loss, grad, pq, span = plain_distill(x[[2, 5]], ids[[2, 5]], t[[2, 5]], 1.0)
    lb, gb = distill_bounds(x, 4, 1.0, loss, grad, pq, span)
    check(out[[2, 5]], loss, lb)
    check(xx.grad[[2, 5]], grad, gb(1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_distill_repeated_ids_and_strides(dtype):
    x, ids, t = make_distill(5, 801, 12, dtype, 13)
    ids[0] = ids[0, 0]                                       # one column twelve times
    ids[1, 5:9] = ids[1, 2]
    ids[2, -1] = ids[2, 0]
    check_distill(x, ids, t, 1.5)
    wide = torch.zeros(5, 1000, dtype=dtype, device="cuda")
    wide[:, 3:804] = x
    check_distill(wide[:, 3:804], ids, t, 1.5)               # rows that start anywhere
    check_distill(x[:, ::2], ids // 2, t, 1.5)               # columns not next to each other
    check_distill(x, ids[:1].expand(5, 12), t[:1].expand(5, 12), 1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 260])
def test_distill_large_offsets_and_lowest_values(rows):
    """softmax does not see a row's offset; a row that is the type's lowest value everywhere is uniform"""
    x, ids, t = make_distill(rows, 700, 5, torch.float32, 17)
    x = (x * 8).round() / 8                                  # (eighths: 5e4 + x is exact)
    x[0] += 5e4
    x[1] -= 5e4
    x[2] = torch.finfo(torch.float32).min
    check_distill(x, ids, t, 0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v,k", [(200, 3001, 9), (193, 20, 3), (300, 9000, 40), (191, 9001, 7), (4, 70001, 64),
                                      (193, 50001, 5), (192, 25000, 8), (200, 70005, 3)])
def test_distill_rows_on_both_sides_of_the_split(dtype, rows, v, k):
    check_distill(*make_distill(rows, v, k, dtype, rows + v + k), 1.25)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x, ids, t = make_distill(3, 50, 4, torch.float32, 18)
    xx = x.detach().requires_grad_()
    g, = torch.autograd.grad(ops.topk_distill_loss(xx * xx, ids, t), xx, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    w = torch.randn(5, 8, device="cuda", requires_grad=True)
    out = ops.embedding(w * w, torch.tensor([1, 2], device="cuda"))
    g, = torch.autograd.grad((out * out).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
def test_distill_k1_is_cross_entropy():
    x, ids, _ = make_distill(40, 1234, 1, torch.float32, 14)
    xx = x.detach().requires_grad_()
    loss = ops.topk_distill_loss(xx, ids, torch.zeros(40, 1, device="cuda"))
    loss.backward()
    x64 = x.double().cpu().requires_grad_()
    want = torch.nn.functional.cross_entropy(x64, ids[:, 0].cpu())
    want.backward()
    assert abs(float(loss) - float(want)) <= U * 200 * 20
    check(xx.grad, x64.grad, x64.grad.abs() * 1e-5 + 1e-9)


@pytest.mark.gpu
def test_distill_gradient_against_differences():
    x, ids, t = make_distill(3, 41, 5, torch.float32, 15)
    xx = x.detach().requires_grad_()
    ops.topk_distill_loss(xx, ids, t, 2.0, reduction="sum").backward()
    for r, c in ((0, int(ids[0, 0])), (1, 7), (2, int(ids[2, 4]))):
        d = torch.zeros(3, 41, dtype=torch.float64)
        d[r, c] = 1e-4
        up, dn = (plain_distill(x.double().cpu() + s * d, ids, t, 2.0)[0].sum() for s in (1, -1))
        # (third derivative of the loss below 1: the central difference is off by at most h^2 / 6, plus the 64-bit rounding)
        assert abs(float(xx.grad[r, c]) - float((up - dn) / 2e-4)) <= 1e-8 + 1e-10 + 100 * U


@pytest.mark.gpu
def test_distill_backward_twice_and_scaled():
    """a kept graph gives the same gradient again, whatever the upstream factors were"""
    x, ids, t = make_distill(33, 3001, 7, torch.float32, 16)
    xx = x.detach().requires_grad_()
    loss = ops.topk_distill_loss(xx, ids, t, 1.0)
    one, = torch.autograd.grad(loss, xx, retain_graph=True)
    keep = one.clone()
    one.zero_()                                              # what the caller does to its gradient stays with the caller
    two, = torch.autograd.grad(loss, xx, torch.tensor(2.0, device="cuda"), retain_graph=True)
    three, = torch.autograd.grad(loss, xx, torch.tensor(1.0, device="cuda"))
    assert torch.equal(two, keep * 2) and torch.equal(three, keep)


@pytest.mark.gpu
def test_distill_empty_batch():
    x = torch.empty(0, 17, device="cuda", requires_grad=True)
    ids, t = torch.empty(0, 3, dtype=torch.int64, device="cuda"), torch.empty(0, 3, device="cuda")
    loss = ops.topk_distill_loss(x, ids, t)
    loss.backward()
    assert float(loss.detach()) == 0.0 and x.grad.shape == (0, 17)
    assert ops.topk_distill_loss(x.detach(), ids, t, reduction="none").shape == (0,)


# ----------------------------------------------------------------------------- microscaled 4 bits
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def plain_mx4(x):
    """-> codes [rows, cols] (0 .. 15), exponents [rows, blocks], values [rows, cols] (64 bits)"""
    x = x.double().cpu()
    rows, cols = x.shape
    blocks = (cols + 31) // 32
    f = torch.zeros(rows, blocks * 32, dtype=torch.float64)
    f[:, :cols] = x
    f = f.view(rows, blocks, 32)
    top = f.abs().amax(2)
    bad = ~torch.isfinite(f).all(2)
    _, e = torch.frexp(torch.where(bad, torch.ones_like(top), top))
    e = torch.where(top == 0, torch.full_like(e, -127), (e - 3).clamp(-127, 127))
    s = torch.ldexp(torch.ones_like(top), e)
    a = torch.where(bad[..., None], torch.zeros_like(f), f).abs() / s[..., None]
    dist = (a.clamp(max=6.0)[..., None] - GRID).abs()
    best = dist.amin(-1, keepdim=True)
    tie = dist == best                                       # two codes at a tie: the even one
    code = torch.where(tie.sum(-1) == 2, (tie & (torch.arange(8) % 2 == 0)).long().argmax(-1), tie.long().argmax(-1))
    value = GRID[code] * s[..., None]
    neg = torch.signbit(f)
    value = torch.where(neg, -value, value)
    value = torch.where(bad[..., None], torch.full_like(value, math.nan), value)
    return (code + 8 * neg).view(rows, -1), torch.where(bad, torch.full_like(e, 128), e), value.view(rows, -1)[:, :cols]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 128), (4, 129), (9, 770), (1000, 256), (3, 1000)])
def test_mx4_quantize(dtype, rows, cols):
    gen = torch.Generator().manual_seed(rows * 10 + cols)
    x = (torch.randn(rows, cols, generator=gen) * torch.exp(3 * torch.randn(rows, 1, generator=gen))).to(dtype)
    check_mx4(x.cuda())


def check_mx4(x):
    q = ops.mx4_quantize(x)
    code, e, value = plain_mx4(x)
    rows, cols = x.shape
    p = (cols + 127) // 128 * 128
    codes = q.codes.cpu().permute(1, 0, 2).reshape(rows, p // 2)
    got = torch.stack([codes & 15, codes >> 4], 2).view(rows, p).long()
    live = torch.repeat_interleave(e != 128, 32, dim=1)[:, :cols]
    assert torch.equal(torch.where(live, got[:, :cols], 0), torch.where(live, code[:, :cols], 0))
    assert int(got[:, cols:].max() if p > cols else 0) == 0                # padded columns are zeros
    blocks = (cols + 31) // 32
    assert torch.equal(q.scales.cpu().permute(1, 0, 2).reshape(rows, p // 32)[:, :blocks].long(), e.long() + 127)
    for dt in (torch.float32, torch.bfloat16):
        check(ops.mx4_dequantize(q, dt), value, 0.0)
    h, t = half_step(torch.float16)
    inside = value.clamp(-65504, 65504)
    v16 = ops.mx4_dequantize(q, torch.float16)
    sel = value.abs() <= 65504
    check(v16.cpu()[sel], value[sel], inside[sel].abs() * h + t)


@pytest.mark.gpu
def test_mx4_quantize_ties_extremes_and_nonfinite():
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 0.2499, 0.2501, -0.25, -5.0, -0.0, 0.0])
    x = torch.zeros(16, 64)
    x[0, :16] = ties
    x[1, :16] = ties * 2.0 ** -126                           # near the smallest scale
    x[2, :16] = ties * 2.0 ** 125                            # the largest exponents
    x[3, :3] = torch.tensor([1e-45, -1e-40, 2.0 ** -128])    # denormals
    x[4, 5] = math.inf
    x[5, 40] = math.nan
    x[6, 0], x[6, 33] = -math.inf, 1.0
    x[7] = torch.finfo(torch.float32).max
    x[8] = torch.finfo(torch.float32).tiny
    x[9, :4] = torch.tensor([4.0, 3.9999998, 4.0000005, -8.0])
    check_mx4(x.cuda())
    check_mx4(x.to(torch.bfloat16).cuda())
    check_mx4(x.to(torch.float16).cuda())


@pytest.mark.gpu
def test_mx4_quantize_strides():
    gen = torch.Generator().manual_seed(8)
    big = torch.randn(30, 333, generator=gen).cuda()
    check_mx4(big[::3, 5:205])
    check_mx4(big.t()[:50])
    check_mx4(big[:1].expand(4, 333))
    check_mx4(torch.randn(20, 264, generator=gen).to(torch.bfloat16).cuda()[:, 8:])
    assert ops.mx4_quantize(big[:0]).codes.shape == (3, 0, 64)


def check_linear(x, w, bias, out_dtype, got=None):
    _, _, xv = plain_mx4(x.reshape(-1, x.size(-1)))
    _, _, wv = plain_mx4(w)
    want = xv @ wv.t()
    mag = xv.nan_to_num(0).abs() @ wv.nan_to_num(0).abs().t()
    if bias is not None:
        want = want + bias.double().cpu()
        mag = mag + bias.double().cpu().abs()
    h, t = half_step(out_dtype)
    if got is None:
        got = ops.mx4_linear(x, ops.mx4_quantize(w), bias=bias, out_dtype=out_dtype)
    assert got.dtype == out_dtype
    # products of two 4-bit values and two powers of two are exact; the sums are fp32 in some order
    check(got.reshape(want.shape), want, want.abs() * h + (x.size(-1) + 4) * U * mag * (1 + h) + t)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 130, 256), (3, 17, 33), (16, 300, 128), (17, 64, 129), (33, 129, 200),
                                   (130, 257, 256), (64, 1000, 768), (300, 70, 1000), (257, 513, 384), (5, 5000, 256),
                                   (129, 128, 2048), (4099, 4100, 1100), (3, 70000, 1025), (33, 5000, 128),
                                   (700, 3000, 100), (200, 1024, 256), (1000, 2049, 250), (8200, 200, 256), (20, 40, 5000),
                                   (32, 65600, 300), (1, 1, 8192), (2, 600, 4000), (40000, 130, 200),
                                   (700, 8200, 256), (1100, 1000, 200), (600, 1040, 500), (300, 544, 100), (2100, 1000, 700),
                                   (4200, 5000, 1100), (3600, 3500, 2000), (500, 700, 8200), (33, 5000, 8192), (64, 30, 4000), (8000, 17, 1100),
                                   (900, 1100, 1030), (40, 129, 1025), (8000, 17, 4097),
                                   (100, 3, 8320), (1000, 1000, 4100)])
@pytest.mark.parametrize("dtype,out", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                       (torch.float16, torch.float32), (torch.bfloat16, torch.float16)])
def test_mx4_linear(m, n, k, dtype, out):
    gen = torch.Generator().manual_seed(m + n + k)
    x = (torch.randn(m, k, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen))).to(dtype).cuda()
    w = (torch.randn(n, k, generator=gen) / math.sqrt(k)).to(dtype).cuda()
    bias = torch.randn(n, generator=gen).cuda() if (m + n) % 2 else None
    check_linear(x, w, bias, out)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,out", [(1100, 130000, 200, torch.float32), (1300, 130008, 400, torch.bfloat16),
                                       (600, 240016, 100, torch.float16), (9000, 20000, 1100, torch.bfloat16)])
def test_mx4_linear_of_huge_results(m, n, k, out):
    """results beyond the caches, rows of every alignment; the product of the held values in 64 bits on the device"""
    gen = torch.Generator().manual_seed(m + n)
    x = (torch.randn(m, k, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen))).cuda()
    w = torch.randn(n, k, generator=gen).cuda()
    bias = torch.randn(n, generator=gen).cuda()
    table = ops.mx4_quantize(w)
    store = torch.full((m + 2, n), 7.0, dtype=out, device="cuda")
    got = ops.mx4_linear(x, table, bias=bias, out_dtype=out)
    h, t = half_step(out)
    xv, wv = ops.mx4_dequantize(ops.mx4_quantize(x)).double(), ops.mx4_dequantize(table).double()
    for lo in range(0, m, 500):
        want = xv[lo:lo + 500] @ wv.t() + bias.double()
        mag = xv[lo:lo + 500].abs() @ wv.abs().t() + bias.double().abs()
        over = (got[lo:lo + 500].double() - want).abs() - (want.abs() * h + (k + 4) * U * mag * (1 + h) + t)
        assert float(over.max()) <= 0
    # through the C entry into the middle of a buffer: nothing beside the rows is written
    a = ops.mx4_quantize(x)
    L.call("bkg_mx4_matmul", a.codes_ptr, a.scales_ptr, m, table.codes_ptr, table.scales_ptr, n, k, bias.data_ptr(),
           store[1].data_ptr(), ops_type(out), n, None, 0, L.stream())
    assert torch.equal(store[1:-1], got) and bool((store[[0, -1]] == 7).all())


def ops_type(dtype):
    return TYPES.index(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [200, 700, 1300, 4200])
@pytest.mark.parametrize("start,ldo", [(0, 1000), (8, 1008), (24, 1024), (3, 1001), (56, 1016)])
def test_mx4_matmul_into_a_view(k, start, ldo):
    """rows of an output with any start and pitch: only the product's places are written"""
    m, n = (1200, 950) if k < 4000 else (650, 950)
    gen = torch.Generator().manual_seed(k + start)
    a, b = ops.mx4_quantize(torch.randn(m, k, generator=gen).cuda()), ops.mx4_quantize(torch.randn(n, k, generator=gen).cuda())
    want = ops.mx4_linear(a, b, out_dtype=torch.bfloat16)
    store = torch.full((m * ldo + start + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(L.lib().bkg_mx4_matmul_workspace_bytes(m, n, k), dtype=torch.uint8, device="cuda")
    L.call("bkg_mx4_matmul", a.codes_ptr, a.scales_ptr, m, b.codes_ptr, b.scales_ptr, n, k, None, store.data_ptr() + 2 * start, 1,
           ldo, L.ptr(ws), ws.numel(), L.stream())
    if ws.numel():
        with pytest.raises(L.HipLibraryError):
            L.call("bkg_mx4_matmul", a.codes_ptr, a.scales_ptr, m, b.codes_ptr, b.scales_ptr, n, k, None,
                   store.data_ptr() + 2 * start, 1, ldo, L.ptr(ws), ws.numel() - 1, L.stream())
    view = store[start:start + m * ldo].view(m, ldo)
    assert torch.equal(view[:, :n], want)                    # (whatever the tiles, the sums run over the panels in order)
    view[:, :n] = 7
    assert bool((store == 7).all())


@pytest.mark.gpu
def test_mx4_linear_forms():
    gen = torch.Generator().manual_seed(21)
    x = torch.randn(2, 3, 96, generator=gen).cuda()
    w = torch.randn(50, 96, generator=gen).cuda()
    table = ops.mx4_quantize(w)
    got = ops.mx4_linear(x, table)
    assert got.shape == (2, 3, 50)
    check_linear(x, w, None, torch.float32, got)
    packed = ops.mx4_linear(ops.mx4_quantize(x.view(6, 96)), table)
    assert torch.equal(packed, got.view(6, 50))
    assert ops.mx4_linear(x[:0], table).shape == (0, 3, 50)
    assert ops.mx4_linear(x[0, 0], table).shape == (50,)
    # block scales of very different sizes along one row, and a NaN block in one row of either operand
    xs = torch.randn(40, 256, generator=gen) * torch.exp2(torch.randint(-30, 30, (40, 8), generator=gen).float()).repeat_interleave(32, 1)
    ws = torch.randn(70, 256, generator=gen) * torch.exp2(torch.randint(-30, 30, (70, 8), generator=gen).float()).repeat_interleave(32, 1)
    check_linear(xs.cuda(), ws.cuda(), None, torch.float32)
    xs[3, 40] = math.nan
    ws[5, 200] = math.inf
    check_linear(xs.cuda(), ws.cuda(), None, torch.float32)


# ----------------------------------------------------------------------------- streams, graphs, a run of them together
@pytest.mark.gpu
def test_entity_ops_on_another_stream():
    x, ids, t = make_distill(20, 3000, 8, torch.float32, 31)
    w = torch.randn(500, 64, generator=torch.Generator().manual_seed(1)).cuda()
    where = torch.randint(0, 500, (9000,), generator=torch.Generator().manual_seed(2)).cuda()
    g = torch.randn(9000, 64, generator=torch.Generator().manual_seed(3)).cuda()
    want = (*run_embedding(w, where, 2.0, None, g), ops.topk_distill_loss(x, ids, t), ops.mx4_linear(w[:30], ops.mx4_quantize(w)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (*run_embedding(w, where, 2.0, None, g), ops.topk_distill_loss(x, ids, t), ops.mx4_linear(w[:30], ops.mx4_quantize(w)))
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def _step(w, ids, tid, tl):
    """queries looked up, scored against every row, distilled: the three operators and the framework's own product"""
    q = ops.embedding(w, ids, scale=0.5)
    logits = ops.linear(q, w)
    return ops.topk_distill_loss(logits, tid, tl, 2.0)


@pytest.mark.gpu
def test_entity_ops_in_a_graph():
    """a training step and a served product captured once and replayed with other inputs equal the eager calls every time"""
    gen = torch.Generator().manual_seed(41)
    w = (0.2 * torch.randn(700, 64, generator=gen)).cuda().requires_grad_()
    ids = torch.randint(0, 700, (9000,), generator=gen).cuda()[:96].contiguous()
    many = torch.randint(0, 700, (9000,), generator=gen).cuda()
    g = torch.randn(9000, 64, generator=gen).cuda()
    tid, tl = torch.randint(0, 700, (96, 6), generator=gen).cuda(), torch.randn(96, 6, generator=gen).cuda()

    def work():
        w.grad = None
        loss = _step(w, ids, tid, tl)
        loss.backward()
        wm = w.detach().requires_grad_()
        ops.embedding(wm, many).backward(g)                  # (the device-wide sort)
        with torch.no_grad():
            y = ops.mx4_linear(w[:50], ops.mx4_quantize(w))
        return loss.detach(), w.grad, wm.grad, y

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            work()
    torch.cuda.current_stream().wait_stream(side)
    w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in range(4):
        gen = torch.Generator().manual_seed(100 + seed)
        with torch.no_grad():
            w.copy_((0.2 * torch.randn(700, 64, generator=gen)).cuda())
            ids.copy_(torch.randint(0, 700, (96,), generator=gen).cuda())
            many.copy_((torch.rand(9000, generator=gen).pow(4) * 700).long().cuda())
            tid.copy_(torch.randint(-1, 700, (96, 6), generator=gen).cuda())
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        ops.note_graph_replay()
        saved = w.grad
        wx = w.detach().clone().requires_grad_()
        loss = _step(wx, ids, tid, tl)
        loss.backward()
        wm = w.detach().requires_grad_()
        ops.embedding(wm, many).backward(g)
        with torch.no_grad():
            y = ops.mx4_linear(w[:50], ops.mx4_quantize(w))
        torch.cuda.synchronize()
        w.grad = saved
        assert torch.equal(got[0], loss.detach()) and torch.equal(got[2], wm.grad) and torch.equal(got[3], y)
        # (the logits' own product splits its inner dimension with atomics in the backward: not bit-equal)
        assert float((got[1] - wx.grad).abs().max()) <= 1e-5 * float(wx.grad.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_gradients_from_tensors_that_hooks_moved(reduction):
    """saved tensors that went to the host and back, and a recomputed step: the same gradients, whatever lies where they were"""
    x, tid, tl = make_distill(9, 5000, 6, torch.bfloat16, 61)
    x, tid, tl = x[:, :4991], tid.clamp(max=4990)[:, ::2], tl[:, ::2]
    w = torch.randn(400, 40, generator=torch.Generator().manual_seed(62)).cuda()
    where = torch.randint(0, 400, (2, 3000), generator=torch.Generator().manual_seed(63)).cuda().t()
    g = torch.randn(3000, 2, 40, generator=torch.Generator().manual_seed(64)).cuda()
    up = torch.rand(9, generator=torch.Generator().manual_seed(65)).cuda()

    def step(how):
        xx, ww = x.detach().clone().requires_grad_(), w.detach().requires_grad_()

        def both(a, b):
            loss = ops.topk_distill_loss(a * 2, tid.clone(), tl.clone(), 2.0, reduction=reduction)
            return (loss * up).sum(), ops.embedding(b * 2, where.clone(), 0.5)
        if how == "host":
            with torch.autograd.graph.save_on_cpu():
                loss, out = both(xx, ww)
        elif how == "again":
            loss, out = torch.utils.checkpoint.checkpoint(both, xx, ww, use_reentrant=False)
        else:
            loss, out = both(xx, ww)
        junk = [torch.full((n,), 7, dtype=torch.int64, device="cuda") for n in (27, 54, 3000, 6000, 6000, 22460)]
        torch.autograd.backward([loss, out], [torch.ones_like(loss), g])
        del junk
        return loss.detach(), out.detach(), xx.grad, ww.grad

    want = step("plain")
    for how in ("host", "again"):
        for a, b in zip(step(how), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_entity_ops_in_two_graphs_at_once():
    """two captured steps replayed side by side on two streams: nothing of one lies in the other's memory"""
    def make(seed):
        gen = torch.Generator().manual_seed(seed)
        w = (0.2 * torch.randn(900, 64, generator=gen)).cuda()
        many = torch.randint(0, 900, (20000,), generator=gen).cuda()
        g = torch.randn(20000, 64, generator=gen).cuda()
        x, tid, tl = make_distill(30, 9000, 6, torch.bfloat16, seed)

        def work():
            wm, xm = w.detach().requires_grad_(), x.detach().requires_grad_()
            out = ops.embedding(wm, many, 3.0)
            out.backward(g)
            loss = ops.topk_distill_loss(xm, tid, tl, 2.0)
            loss.backward()
            return out.detach(), wm.grad, loss.detach(), xm.grad, ops.mx4_linear(w[:50], ops.mx4_quantize(w))
        return work

    works, graphs, outs, wants = [make(51), make(52)], [], [], []
    for work in works:
        wants.append([o.clone() for o in work()])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(work())
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for out in outs:
            for o in out:
                o.zero_()
        for s, graph in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        again = works[0]()
        torch.cuda.synchronize()
        for got, want in list(zip(outs, wants)) + [(again, wants[0])]:
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_embedding_beyond_32_bits():
    v, d = 4500000, 512                                      # 2.3e9 values, 4.6 GB
    w = torch.empty(v, d, dtype=torch.bfloat16, device="cuda").normal_()
    ids = torch.tensor([v - 1, 0, v - 2, v - 1, 4194303, 4194304, 4194305, v, -1, v - 1], device="cuda")
    g = torch.randn(10, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    out, dw = run_embedding(w, ids, 1.0, None, g)
    assert torch.equal(out[[7, 8]], torch.zeros(2, d, dtype=torch.bfloat16, device="cuda"))
    live = ids[[0, 1, 2, 4, 5, 6]]
    assert torch.equal(out[[0, 1, 2, 4, 5, 6]], w[live]) and torch.equal(out[3], out[0]) and torch.equal(out[9], out[0])
    small = torch.tensor([0, 1, 2, 0, 3, 4, 5, 9, 9, 0])     # the same with the live rows side by side
    want, mag, cnt = plain_embedding_grad(g, small, 6, 1.0, None)
    h, t = half_step(torch.bfloat16)
    check(dw[live], want, want.abs() * h + (cnt[:, None] + 4) * U * mag * (1 + h) + t)
    dw[live] = 0
    assert not bool(dw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 3000])
def test_embedding_of_as_many_rows_as_there_may_be(n):
    v = 2 ** 31 - 1
    w = torch.zeros(v, 1, dtype=torch.bfloat16, device="cuda")
    live = torch.tensor([0, 1, 2097151, 2097152, 2 ** 30, 2 ** 30 + 1, v - 2, v - 1], device="cuda")
    w[live, 0] = torch.arange(1, 9, device="cuda").bfloat16()
    which = torch.randint(0, 9, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    ids = torch.cat([live, live.new_tensor([v])])[which]                  # (the last: outside)
    g = torch.ones(n, 1, dtype=torch.bfloat16, device="cuda")
    out, dw = run_embedding(w, ids, 2.0, None, g)
    assert torch.equal(out[:, 0], torch.where(which < 8, 2.0 * (which + 1), 0.0).bfloat16())
    assert torch.equal(dw[live, 0], (2.0 * torch.bincount(which, minlength=9)[:8]).bfloat16())
    dw[live] = 0
    assert not bool(dw.any())
    with pytest.raises(ValueError):
        ops.embedding(w.new_empty(1, 1).expand(v + 1, 1), ids)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v", [(1100, 2000003), (3, 800000001)])
def test_distill_beyond_32_bits(rows, v):
    x = torch.empty(rows, v, dtype=torch.bfloat16, device="cuda").normal_()
    gen = torch.Generator().manual_seed(2)
    ids, tl = torch.randint(0, v, (rows, 5), generator=gen).cuda(), torch.randn(rows, 5, generator=gen).cuda()
    ids[-1, 0] = v - 1
    xx = x.requires_grad_()
    loss = ops.topk_distill_loss(xx, ids, tl, 1.0, reduction="sum")
    loss.backward()
    losses = ops.topk_distill_loss(x.detach(), ids, tl, 1.0, reduction="none")
    row = x.detach()[-1].double()                            # the last row, in 64 bits on the device
    lp = row - torch.logsumexp(row, 0)
    lq = torch.log_softmax(tl[-1].double(), 0)
    want = float((lq.exp() * (lq - lp[ids[-1]])).sum())
    span = float(row.max() - row.min())
    err = U * (3 * span + v / 256 + 42)                      # (distill_bounds; up to v / 256 terms in a thread's chain)
    assert abs(float(losses[-1]) - want) <= err * (4 + 2 * span + 2 * math.log(v + 1))
    p = lp.exp()
    pq = p.clone()
    p.index_add_(0, ids[-1], -lq.exp())
    pq.index_add_(0, ids[-1], lq.exp())
    h, t = half_step(torch.bfloat16)
    over = (xx.grad[-1].double() - p).abs() - (p.abs() * (h + 4 * U) + 2 * err * pq * (1 + h) + t)
    assert float(over.max()) <= 0


@pytest.mark.gpu
def test_mx4_beyond_32_bits():
    n, k = 34000001, 200                                     # 4.4 GB of codes, outputs beyond 2^31 values
    w = torch.empty(n, k, dtype=torch.bfloat16, device="cuda").normal_()
    table = ops.mx4_quantize(w)
    tail = w[-300:].clone()
    del w
    want = ops.mx4_quantize(tail)
    assert torch.equal(table.codes[:, -300:], want.codes) and torch.equal(table.scales[:, -300:], want.scales)
    x = torch.randn(70, k, generator=torch.Generator().manual_seed(3)).cuda()
    for m in (2, 70):
        got = ops.mx4_linear(x[:m], table, out_dtype=torch.bfloat16)
        check_linear(x[:m], tail, None, torch.bfloat16, got[:, -300:])
        del got
    values = ops.mx4_dequantize(table, torch.bfloat16)
    assert torch.equal(values[-300:], ops.mx4_dequantize(want, torch.bfloat16))


# ----------------------------------------------------------------------------- refusals (no GPU needed)
def test_entity_ops_refuse_cpu_tensors():
    w = torch.randn(4, 8)
    with pytest.raises(L.HipLibraryError):
        ops.embedding(w, torch.tensor([1]))
    with pytest.raises(L.HipLibraryError):
        ops.topk_distill_loss(w, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))
    with pytest.raises(L.HipLibraryError):
        ops.mx4_quantize(w)
    table = ops.Mx4Table(torch.zeros(1, 4, 64, dtype=torch.uint8), torch.zeros(1, 4, 4, dtype=torch.uint8), (4, 8))
    with pytest.raises(L.HipLibraryError):
        ops.mx4_linear(w, table)
    with pytest.raises(L.HipLibraryError):
        ops.mx4_dequantize(table)


def test_entity_ops_refuse_bad_arguments():
    w, ids = torch.randn(4, 8), torch.tensor([1])
    with pytest.raises(ValueError):
        ops.embedding(torch.randn(4), ids)
    with pytest.raises(TypeError):
        ops.embedding(w.double(), ids)
    with pytest.raises(TypeError):
        ops.embedding(w, ids.float())
    tid, tl = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2)
    with pytest.raises(ValueError):
        ops.topk_distill_loss(w, tid[:3], tl[:3])
    with pytest.raises(ValueError):
        ops.topk_distill_loss(w, tid, tl[:, :1])
    with pytest.raises(TypeError):
        ops.topk_distill_loss(w.double(), tid, tl)
    with pytest.raises(TypeError):
        ops.topk_distill_loss(w, tid.float(), tl)
    with pytest.raises(ValueError):
        ops.mx4_quantize(torch.randn(4))
    with pytest.raises(ValueError):
        ops.mx4_quantize(torch.randn(4, 0))
    with pytest.raises(TypeError):
        ops.mx4_quantize(w.double())
    with pytest.raises(TypeError):
        ops.mx4_linear(w, w)
    with pytest.raises(TypeError):
        ops.mx4_dequantize(w)
    with pytest.raises(ValueError):
        ops.Mx4Table(torch.zeros(1, 4, 63, dtype=torch.uint8), torch.zeros(1, 4, 4, dtype=torch.uint8), (4, 8))


@pytest.mark.gpu
def test_entity_ops_refuse_bad_calls():
    w, ids = torch.randn(4, 8).cuda(), torch.tensor([1]).cuda()
    tid, tl = torch.zeros(4, 2, dtype=torch.int64).cuda(), torch.zeros(4, 2).cuda()
    with pytest.raises(ValueError):
        ops.embedding(w, ids, padding_idx=4)
    with pytest.raises(L.HipLibraryError):
        ops.embedding(w, ids.cpu())
    many = torch.zeros(2 ** 22, 1, device="cuda")
    with pytest.raises(ValueError):
        ops.topk_distill_loss(many, many.long(), many)
    for temp in (0.0, -1.0, math.inf, math.nan, 1e-30, 1e30):
        with pytest.raises(ValueError):
            ops.topk_distill_loss(w, tid, tl, temp)
    with pytest.raises(ValueError):
        ops.topk_distill_loss(w, tid, tl, reduction="mean")
    with pytest.raises(ValueError):
        ops.topk_distill_loss(w, tid, tl.requires_grad_())
    with pytest.raises(ValueError):
        ops.topk_distill_loss(w, torch.zeros(4, 1025, dtype=torch.int64).cuda(), torch.zeros(4, 1025).cuda())
    with pytest.raises(ValueError):
        ops.topk_distill_loss(w, tid[:, :0], tl.detach()[:, :0])
    with pytest.raises(ValueError):
        ops.topk_distill_loss(w[:, :0], tid, tl.detach())
    table = ops.mx4_quantize(torch.randn(5, 8).cuda())
    with pytest.raises(ValueError):
        ops.mx4_linear(w.requires_grad_(), table)
    w = w.detach()
    with pytest.raises(ValueError):
        ops.mx4_linear(w[:, :7], table)
    with pytest.raises(ValueError):
        ops.mx4_linear(w, table, bias=torch.zeros(4).cuda())
    with pytest.raises(TypeError):
        ops.mx4_linear(w, table, out_dtype=torch.float64)
