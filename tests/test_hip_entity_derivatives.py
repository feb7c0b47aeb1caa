"""What the entity-prediction operators do with derivatives they do not compute: they refuse, also where a plain call would
record nothing."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from biomedkg_amd import _lib as L
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


@pytest.mark.parametrize("packed", [False, True])
def test_product_refuses_a_bias_that_requires_a_gradient(packed):
    x, table = torch.randn(3, 8), ops.Mx4Table(torch.zeros(1, 6, 64, dtype=torch.uint8), torch.zeros(1, 6, 4, dtype=torch.uint8), (6, 8))
    if packed:
        x = ops.Mx4Table(torch.zeros(1, 3, 64, dtype=torch.uint8), torch.zeros(1, 3, 4, dtype=torch.uint8), (3, 8))
    bias = torch.zeros(6, requires_grad=True)
    with pytest.raises(ValueError, match="without a gradient"):
        ops.mx4_linear(x, table, bias=bias)
    with torch.no_grad(), pytest.raises(L.HipLibraryError):      # (as far as the tensors' device)
        ops.mx4_linear(x, table, bias=bias)


@pytest.mark.gpu
def test_packed_product_and_a_bias_that_requires_a_gradient():
    gen = torch.Generator().manual_seed(3)
    x, table = ops.mx4_quantize(torch.randn(3, 8, generator=gen).cuda()), ops.mx4_quantize(torch.randn(6, 8, generator=gen).cuda())
    bias = torch.randn(6, generator=gen).cuda().requires_grad_()
    with pytest.raises(ValueError):
        ops.mx4_linear(x, table, bias=bias)
    with torch.no_grad():
        assert torch.equal(ops.mx4_linear(x, table, bias=bias), ops.mx4_linear(x, table, bias=bias.detach()))
