"""The one-pass walk over node-sorted incidences through its C entry, with and without scores (csrc/kge_onepass_mx.hip), against
64 bits: lists of every length, nodes without entries, node counts that are no multiple of four."""
import pytest
import torch

from biomedkg_amd import _lib as L

U, H, D = 2.0 ** -24, 2.0 ** -8, 256


def walk(z, rel, rowptr2, packed, perm, t, label, scores):
    n, r = z.size(0), rel.size(0)
    lib = L.lib()
    assert lib.bkg_kge_onepass_mx_ok(D, 1, r)
    blocks = lib.bkg_kge_onepass_mx_blocks(n)
    score = torch.full((t,), 7.0, device="cuda") if scores else None
    loss = torch.full((4 * blocks,), 7.0, device="cuda")
    dz = torch.full((n, D), 7.0, device="cuda")
    drel = torch.full((blocks, 32, D), 7.0, device="cuda")
    L.call("bkg_kge_onepass_mx_f32", L.ptr(z), z.stride(0), n, L.ptr(rel), rel.stride(0), r, L.ptr(rowptr2), L.ptr(packed),
           L.ptr(perm) if scores else None, 2 * t, label, 1.0 / t, L.ptr(score), L.ptr(loss), L.ptr(dz), dz.stride(0),
           L.ptr(drel), blocks, L.stream())
    return score, loss, dz, drel


@pytest.mark.gpu
@pytest.mark.parametrize("n,r,t,label,skew", [(1, 1, 1, 0.0, 1), (5, 3, 7, 1.0, 1), (333, 30, 5000, 0.0, 1), (4, 32, 300, 0.0, 1),
                                              (20001, 17, 9000, 1.0, 1), (1000, 30, 40000, 0.0, 6)])
def test_walk_with_and_without_scores(n, r, t, label, skew):
    gen = torch.Generator().manual_seed(n + t)
    head, tail = ((torch.rand(t, generator=gen).pow(skew) * n).long().clamp_(max=n - 1) for _ in range(2))
    kind = torch.randint(0, r, (t,), generator=gen)
    z, rel = (0.4 * torch.randn(n, D, generator=gen)).bfloat16(), 0.4 * torch.randn(r, D, generator=gen)
    key = torch.cat([2 * head, 2 * tail + 1])
    perm = torch.argsort(key, stable=True)
    other, kinds = torch.cat([tail, head])[perm], torch.cat([kind, kind])[perm]
    rowptr2 = torch.searchsorted(key[perm].contiguous(), torch.arange(2 * n + 1)).int().cuda()
    packed = (other | (kinds << 24)).int().cuda()
    args = (z.cuda(), rel.cuda(), rowptr2, packed, perm.int().cuda(), t, label)
    none, loss, dz, drel = walk(*args, False)
    score, loss_s, dz_s, drel_s = walk(*args, True)
    assert none is None
    for a, b in ((loss, loss_s), (dz, dz_s), (drel, drel_s)):           # (the scores are only written: the rest is the same)
        assert torch.equal(a, b)

    z64, r64 = z.double(), rel.double()
    zh, zt, rk = z64[head], z64[tail], r64[kind]
    s = (zh * rk * zt).sum(1)
    mag = (zh * rk * zt).abs().sum(1)
    s_err = (D + 8) * U * mag                                            # a 256-term fp32 sum of rounded products
    assert bool(((score.double().cpu() - s).abs() <= s_err).all())
    g = torch.sigmoid(s) - label
    g_err = 0.25 * s_err + 16 * U                                        # (the sigmoid's slope; exp2, reciprocal, a few roundings)
    each = torch.nn.functional.softplus(s) - s * label
    assert abs(float(loss.double().sum()) - float(each.sum())) <= float((s_err + (t + 16) * U * (each.abs() + 1)).sum())
    length = torch.bincount(torch.cat([head, tail]), minlength=n).double()[:, None]
    want, bound, size = (torch.zeros(n, D, dtype=torch.float64) for _ in range(3))
    for node, o in ((head, zt), (tail, zh)):
        want.index_add_(0, node, g[:, None] * rk * o)
        bound.index_add_(0, node, g_err[:, None] * (rk * o).abs())
        size.index_add_(0, node, (g[:, None] * rk * o).abs())
    over = (dz.double().cpu() - want / t).abs() - (bound + (length + 8) * U * size) / t
    assert float(over.max()) <= 1e-30
    # the relations' sums: products of bf16 operands (half a step of g z o each), fp32 sums
    want, bound, size = (torch.zeros(32, D, dtype=torch.float64) for _ in range(3))
    want.index_add_(0, kind, g[:, None] * zh * zt)
    bound.index_add_(0, kind, g_err[:, None] * (zh * zt).abs())
    size.index_add_(0, kind, (g[:, None] * zh * zt).abs())
    over = (drel.double().sum(0).cpu() - want).abs() - ((bound + (H + (t + 8) * U) * size) * (1 + H) + 1e-30)
    assert float(over.max()) <= 0
