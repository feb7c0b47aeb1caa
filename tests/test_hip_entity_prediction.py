"""Entity prediction through the model's own surface: ``DistMult.entity_logits``, ``KGEModule.distillation_loss`` /
``top_entities`` / ``set_teacher`` and the training entry point that uses them, against 64-bit autograd on the CPU."""
import os

import pytest
import torch

from biomedkg_amd import ops
from biomedkg_amd.kge_module import KGEModule

U = 2.0 ** -24


def module(dim=32, decoder="dismult", relations=5, seed=0):
    torch.manual_seed(seed)
    return KGEModule("rgcn", decoder, dim, dim, dim, 2, relations, 2, "cosine", 1e-3, 0.2, "none", 2, "random")


class Batch:
    pass


def batch(n=300, e=2500, dim=32, relations=5, seed=1):
    gen = torch.Generator().manual_seed(seed)
    b = Batch()
    b.x = torch.randn(n, dim, generator=gen).cuda()
    b.edge_index = torch.randint(0, n, (2, e), generator=gen).cuda()
    b.edge_type = torch.randint(0, relations, (e,), generator=gen).cuda()
    return b


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,q,k,temp", [(700, 64, 40, 8, 2.0), (5000, 256, 128, 10, 1.0), (37, 20, 3, 37, 0.5)])
def test_distillation_loss_and_gradients(n, d, q, k, temp):
    gen = torch.Generator().manual_seed(n)
    m = module(d).cuda()
    z = (torch.randn(n, d, generator=gen) / d ** 0.25).cuda().requires_grad_()
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

    # logits are within eps of the exact ones (a d-term fp32 product of a rounded q); p and the loss follow
    mag = qr.detach().abs() @ z64.detach().abs().t()
    eps = (d + 8) * U * float(mag.max())
    kappa = 4 * eps / temp + U * (n + q + d + 2 * k + 64 + 3 * float(logits.detach().abs().max()) / temp)
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
def test_top_entities_exact_and_packed():
    gen = torch.Generator().manual_seed(3)
    m = module(48).cuda()
    z = torch.randn(900, 48, generator=gen).cuda()
    anchor, rel = torch.randint(0, 900, (30,), generator=gen).cuda(), torch.randint(0, 5, (30,), generator=gen).cuda()
    q = z[anchor] * m.model.decoder.rel_emb.detach()[rel]
    ids, scores = m.top_entities(z, anchor, rel, 7)
    full = q.double() @ z.double().t()
    want, _ = torch.topk(full, 7, dim=1)
    bound = 64 * U * float((q.double().abs() @ z.double().abs().t()).max())
    assert float((scores - want).abs().max()) <= bound
    assert float((full.gather(1, ids) - want).abs().max()) <= bound
    table = ops.mx4_quantize(z)
    ids4, scores4 = m.top_entities(z, anchor, rel, 7, table=table)
    packed = ops.mx4_dequantize(ops.mx4_quantize(q)).double() @ ops.mx4_dequantize(table).double().t()
    want4, _ = torch.topk(packed, 7, dim=1)
    assert float((scores4 - want4).abs().max()) <= bound * 4
    assert float((packed.gather(1, ids4) - want4).abs().max()) <= bound * 4
    assert m.top_entities(z[:4], torch.zeros(2, dtype=torch.int64, device="cuda"), rel[:2], 10)[0].shape == (2, 4)


@pytest.mark.gpu
def test_training_step_with_a_teacher():
    from biomedkg_amd import rand as R
    b = batch()
    student, teacher = module(seed=5).cuda().train(), module(seed=6)
    names = set(student.state_dict())
    student.set_teacher(teacher, k=6, temperature=2.0, weight=0.5, queries=32)
    assert set(student.state_dict()) == names and student.has_teacher
    assert len(list(student.parameters())) == len(list(module().parameters()))
    seen = []
    orig = student._distillation_term
    student._distillation_term = lambda *a: seen.append(orig(*a)) or seen[-1]
    R.reseed_default(7)
    torch.manual_seed(7)
    with_teacher = student.training_step(b)
    with_teacher.backward()
    assert len(seen) == 1 and float(seen[0].detach()) > 0
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in student.model.parameters())
    assert all(p.grad is None for p in teacher.parameters()) and not teacher.training
    student.set_teacher(None)
    R.reseed_default(7)
    torch.manual_seed(7)
    alone = student.training_step(b)
    assert abs(float(with_teacher.detach() - seen[0].detach() - alone.detach())) <= 1e-5 * float(with_teacher.detach().abs())


@pytest.mark.gpu
def test_teacher_of_another_width_and_refusals():
    b = batch()
    wide = module(dim=64)
    b.x = torch.randn(300, 64, device="cuda")
    student = KGEModule("rgcn", "dismult", 64, 32, 32, 2, 5, 2, "cosine", 1e-3, 0.2, "none", 1, "random").cuda().train()
    student.set_teacher(wide, k=5)
    student.training_step(b).backward()
    with pytest.raises(NotImplementedError):
        student.set_teacher(module(decoder="transe"))
    with pytest.raises(NotImplementedError):
        module(decoder="transe").set_teacher(module())
    with pytest.raises(ValueError):
        student.set_teacher(module(), k=0)
    from biomedkg_amd.sampled import SaintGraphedKge
    with pytest.raises(ValueError):
        SaintGraphedKge(student, b.x, b.edge_index, b.edge_type, 8, 4, None)


def test_set_teacher_refuses():
    student = module()
    for bad in (dict(k=0), dict(k=1025), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=1e-30),
                dict(queries=0)):
        with pytest.raises(ValueError):
            student.set_teacher(module(), **bad)
    with pytest.raises(ValueError):
        student.set_teacher(student)
    with pytest.raises(ValueError):
        student.set_teacher(module(relations=4))
    assert not student.has_teacher and all(p.requires_grad for p in student.parameters())


@pytest.mark.gpu
@pytest.mark.parametrize("sampler", ["full", "device"])
def test_train_kge_distils_from_a_checkpoint(tmp_path, sampler):
    import train_kge
    common = ["devices=[0]", "data=synthetic", f"data.sampler={sampler}", "data.num_nodes=1000", "data.num_edges=12000",
              "data.embed_dim=32", "data.batch_size=32", "data.steps_per_epoch=4", "model.in_dim=32", "model.hidden_dim=32",
              "neg_ratio=1", "epochs=1", "val_every_epoch=1"]
    train_kge.main(common + ["model.out_dim=32", f"ckpt_dir={tmp_path}/teacher"])
    ckpt = [os.path.join(d, f) for d, _, fs in os.walk(f"{tmp_path}/teacher") for f in fs if f == "last.ckpt"][0]
    out = train_kge.main(common + ["model.out_dim=16", f"ckpt_dir={tmp_path}/student", f"teacher_path={ckpt}", "teacher_k=5",
                                   "teacher_temperature=2.0"])
    assert any(k.startswith("test_AUROC") for k in out[0])
