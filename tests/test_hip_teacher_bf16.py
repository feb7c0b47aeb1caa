"""Distillation from a teacher in bf16 mode (products of bf16 operands, fp32 sums), against 64 bits."""
import pytest
import torch

from biomedkg_amd import ops
from biomedkg_amd import rand as R
from biomedkg_amd.kge_module import KGEModule

U, H = 2.0 ** -24, 2.0 ** -8


def module(dim, seed):
    torch.manual_seed(seed)
    return KGEModule("rgcn", "dismult", dim, dim, dim, 2, 5, 2, "cosine", 1e-3, 0.2, "none", 2, "random").cuda()


class Batch:
    pass


def batch(n, e, dim):
    gen = torch.Generator().manual_seed(n + e)
    b = Batch()
    b.x = torch.randn(n, dim, generator=gen).cuda()
    b.edge_index = torch.randint(0, n, (2, e), generator=gen).cuda()
    b.edge_type = torch.randint(0, 5, (e,), generator=gen).cuda()
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,q,k,temp", [(700, 64, 40, 8, 2.0), (5000, 256, 256, 10, 2.0), (4999, 256, 300, 10, 4.0), (37, 20, 3, 37, 4.0)])
def test_loss_and_gradients(n, d, q, k, temp):
    ops.set_matmul_precision("bf16")
    gen = torch.Generator().manual_seed(n)
    m = module(d, 1)
    z = (torch.randn(n, d, generator=gen) / d ** 0.5).cuda().requires_grad_()
    anchor, rel = torch.randint(0, n, (q,), generator=gen).cuda(), torch.randint(0, 5, (q,), generator=gen).cuda()
    ids = torch.stack([torch.randperm(n, generator=gen)[:k] for _ in range(q)]).cuda()
    ids[0] = -1
    t = torch.randn(q, k, generator=gen).cuda()
    loss = m.distillation_loss(z, anchor, rel, ids, t, temp)
    loss.backward()
    rel_emb = m.model.decoder.rel_emb

    z64, r64 = z.detach().double().cpu().requires_grad_(), rel_emb.detach().double().cpu().requires_grad_()
    a, r, i = anchor.cpu(), rel.cpu(), ids.cpu()
    qr = z64[a] * r64[r]
    logits = qr @ z64.t()
    use = i[:, 0] >= 0
    lp = torch.log_softmax(logits / temp, 1)
    tq = torch.softmax(t.double().cpu() / temp, 1)
    row = (tq * (tq.log() - lp.gather(1, i.clamp(min=0)))).sum(1) * temp * temp
    want = torch.where(use, row, torch.zeros(())).sum() / q
    want.backward()

    # logits: a d-term fp32 sum of products of operands that are half a bf16 step off each; the gradients' products round theirs too
    mag = qr.detach().abs() @ z64.detach().abs().t()
    eps = (2 * H + H * H + (d + 8) * U) * float(mag.max())
    kappa = 4 * eps / temp + 2 * H + H * H + U * (n + q + d + 2 * k + 64 + 3 * float(logits.detach().abs().max()) / temp)
    assert abs(float(loss.detach()) - float(want.detach())) <= temp * temp * kappa * (4 + float(row.detach().abs().max()))
    g = lp.detach().exp()
    g.scatter_add_(1, i.clamp(min=0), tq)
    g = torch.where(use[:, None], g, torch.zeros(())) * temp / q
    dq = g @ z64.detach().abs()
    bz = g.t() @ qr.detach().abs()
    bz.index_add_(0, a, dq * r64.detach().abs()[r])
    br = torch.zeros_like(r64).index_add_(0, r, dq * z64.detach().abs()[a])
    for got, ref, bound in ((z.grad, z64.grad, bz), (rel_emb.grad, r64.grad, br)):
        over = (got.double().cpu() - ref).abs() - kappa * bound - 1e-12
        assert float(over.max()) <= 0, (float(over.max()), kappa)


@pytest.mark.gpu
@pytest.mark.parametrize("n,e,dim", [(300, 2500, 32), (5000, 40000, 256)])
def test_training_steps(n, e, dim):
    """the step's loss is the reference's loss plus the distillation term, and every parameter gets a finite gradient; twice, so
    that the second step meets what the first has cached"""
    ops.set_matmul_precision("bf16")
    b, student = batch(n, e, dim), module(dim, 5).train()
    student.set_teacher(module(dim, 6), k=6, temperature=2.0, weight=0.5, queries=32)
    seen = []
    term = student._distillation_term
    student._distillation_term = lambda *a: seen.append(term(*a)) or seen[-1]

    def step():
        R.reseed_default(7)
        torch.manual_seed(7)
        student.zero_grad()
        loss = student.training_step(b)
        loss.backward()
        torch.cuda.synchronize()
        return float(loss.detach())

    both = [step(), step()]
    assert len(seen) == 2 and all(float(s.detach()) > 0 for s in seen)
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in student.model.parameters())
    student.set_teacher(None)
    alone = step()
    for loss, s in zip(both, seen):
        assert abs(loss - float(s.detach()) - alone) <= 1e-5 * abs(loss)
