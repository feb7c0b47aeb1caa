"""``ops.topk_distill_loss`` at the ends of the types' ranges, against 64 bits."""
import pytest
import torch

from biomedkg_amd import ops

U = 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("temp", [0.25, 1.0])
@pytest.mark.parametrize("rows,v,k", [(3, 700, 6), (200, 700, 6), (191, 5000, 1024), (192, 5000, 1024), (2, 70001, 3), (192, 70001, 3)])
def test_teacher_entries_on_logits_of_the_lowest_value(dtype, temp, rows, v, k):
    """several of a row's teacher entries lie on logits masked with the type's lowest value: their losses are huge and finite,
    whichever kernel takes the row"""
    gen = torch.Generator().manual_seed(rows + v + k)
    x = (3 * torch.randn(rows, v, generator=gen)).to(dtype)
    ids = torch.stack([torch.randperm(v, generator=gen)[:k] for _ in range(rows)])
    t = 2 * torch.randn(rows, k, generator=gen)
    masked = k // 2 if k > 3 else 2
    x.scatter_(1, ids[:, :masked], torch.finfo(dtype).min)
    z, tt = x.double() / temp, t.double() / temp
    log_p, log_q = torch.log_softmax(z, 1), torch.log_softmax(tt, 1)
    want = temp * temp * (log_q.exp() * (log_q - log_p.gather(1, ids))).sum(1)
    assert float(want.max()) < torch.finfo(torch.float32).max
    got = ops.topk_distill_loss(x.cuda(), ids.cuda(), t.cuda(), temp, reduction="none").double().cpu()
    # The sum over the masked entries decides: its weights q are off by 3 u of their exponent's range, 2 u of the exponential and
    # (k / 64 + 16) u of the sums they are divided by and added in; the rest of the loss by u of ln s, ln ts and the sums behind them.
    span = float((tt.amax(1) - tt.amin(1)).max())
    rel = U * (3 * span + k / 32 + 40)
    rest = temp * temp * U * 64 * (v / 256 + k + 64)
    over = (got - want).abs() - (rel * want.abs() + rest)
    assert bool(torch.isfinite(got).all()) and float(over.max()) <= 0, float(over.max())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2, 200])
def test_a_masked_entry_without_weight_adds_nothing(rows):
    """an entry whose share of the teacher underflows to zero, on a logit of the lowest value and on one of -inf"""
    x = torch.zeros(rows, 50)
    x[:, 0], x[:, 1] = torch.finfo(torch.float32).min, -float("inf")
    ids, t = torch.tensor([[2, 0, 1]]).expand(rows, 3), torch.tensor([[0.0, -500.0, -500.0]]).expand(rows, 3)
    got = ops.topk_distill_loss(x.cuda(), ids.cuda(), t.cuda(), 1.0, reduction="none").double().cpu()
    want = torch.log(torch.tensor(48.0, dtype=torch.float64))
    assert float((got - want).abs().max()) <= 64 * U * float(want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v", [(1100, 2000003), (3, 800000001)])
def test_beyond_32_bits_no_column_is_left_out(rows, v):
    """the loss and the gradient's mass of logits with more than 2^31 values, to the accuracy of the sums as they are cut: a block
    of 1024 threads for a row, or (few rows) ceil(2048 / rows) blocks of 256"""
    gen = torch.Generator().manual_seed(4)
    x = torch.empty(rows, v, dtype=torch.bfloat16, device="cuda").normal_()
    k = 5
    ids, tl = torch.randint(0, v, (rows, k), generator=gen).cuda(), torch.randn(rows, k, generator=gen).cuda()
    ids[-1, 0] = v - 1
    chain = v / 1024 if rows >= 192 else v / (256 * -(-2048 // rows))
    losses = ops.topk_distill_loss(x, ids, tl, 1.0, reduction="none")
    xx = x.requires_grad_()
    ops.topk_distill_loss(xx, ids, tl, 1.0, reduction="sum").backward()
    for r in (0, rows - 1):
        row = x.detach()[r].double()
        lse = torch.logsumexp(row, 0)
        lq = torch.log_softmax(tl[r].double(), 0)
        want = float((lq.exp() * (lq - (row[ids[r]] - lse))).sum())
        span = float(row.max() - row.min())
        # An exponential is off by 3 u of its argument's range and 2 u; a thread's chain adds u per term, its rescaling when a
        # larger logit comes and the joins of threads, waves and blocks a few u each (64 in all), the teacher's sums 2 k u.
        err = U * (3 * span + chain + 2 * k + 64)
        assert err < 1e-3
        assert abs(float(losses[r]) - want) <= err + U * 8 * (span + 8 + abs(want))
        p = (row - lse).exp()
        pq = p.clone()
        p.index_add_(0, ids[r], -lq.exp())
        pq.index_add_(0, ids[r], lq.exp())
        over = (xx.grad[r].double() - p).abs() - (p.abs() * (2.0 ** -8 + 4 * U) + 2 * err * pq * (1 + 2.0 ** -8) + 2.0 ** -134)
        assert float(over.max()) <= 0
        del row, p, pq, over
