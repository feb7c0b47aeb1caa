"""What the entity-prediction operators do with derivatives they do not compute: they refuse, also where a plain call would
record nothing."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from biomedkg_amd import ops


def _calls(device):
    """name -> a call on plain tensors of `device` with one of them replaced by a dual tensor"""
    gen = torch.Generator().manual_seed(1)
    w, x = torch.randn(6, 8, generator=gen).to(device), torch.randn(3, 8, generator=gen).to(device)
    ids, tid = torch.tensor([1, 4], device=device), torch.zeros(3, 2, dtype=torch.int64, device=device)
    tl, bias = torch.zeros(3, 2, device=device), torch.zeros(6, device=device)

    def packed(rows):
        return ops.Mx4Table(torch.zeros(1, rows, 64, dtype=torch.uint8, device=device),
                            torch.full((1, rows, 4), 127, dtype=torch.uint8, device=device), (rows, 8))

    def dual(t):
        return fwad.make_dual(t, torch.ones_like(t))

    return {
        "embedding": lambda: ops.embedding(dual(w), ids),
        "loss": lambda: ops.topk_distill_loss(dual(x), tid, tl),
        "loss per row": lambda: ops.topk_distill_loss(dual(x), tid, tl, reduction="none"),
        "loss teacher": lambda: ops.topk_distill_loss(x, tid, dual(tl)),
        "product": lambda: ops.mx4_linear(dual(x), packed(6)),
        "product bias": lambda: ops.mx4_linear(x, packed(6), bias=dual(bias)),
        "packed product bias": lambda: ops.mx4_linear(packed(3), packed(6), bias=dual(bias)),
    }


NAMES = list(_calls("cpu"))


def check_refusal(call):
    with fwad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                call()


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    check_refusal(_calls("cpu")[name])


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused_on_the_device(name):
    check_refusal(_calls("cuda")[name])


@pytest.mark.gpu
def test_plain_tensors_inside_a_dual_level():
    gen = torch.Generator().manual_seed(2)
    w, ids = torch.randn(6, 8, generator=gen).cuda(), torch.tensor([1, 4]).cuda()
    want = ops.embedding(w, ids)
    with fwad.dual_level():
        assert torch.equal(ops.embedding(w, ids), want)
