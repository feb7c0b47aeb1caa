"""The settings of a distillation run reach ``KGEModule.set_teacher`` as they were given (``train_kge.py teacher_*=``)."""
import os

import pytest
import torch

import train_kge
from biomedkg_amd.config import compose
from biomedkg_amd.kge_module import KGEModule

CFG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "configs")
DATA = ["data=synthetic", "data.num_nodes=300", "data.num_edges=2000", "data.embed_dim=16", "model.in_dim=16", "model.hidden_dim=16",
        "model.out_dim=16", "neg_ratio=1"]


@pytest.fixture(scope="module")
def checkpoint(tmp_path_factory):
    from biomedkg_amd.trainer import Trainer
    _, teacher = train_kge.build(compose(CFG, "kge", DATA), "kge")
    path = str(tmp_path_factory.mktemp("teacher") / "last.ckpt")
    Trainer(max_epochs=1).save_checkpoint(teacher, path)
    return path


def built(checkpoint, *settings):
    return train_kge.build(compose(CFG, "kge", DATA + [f"teacher_path={checkpoint}", *settings]), "kge")[1]._teacher


def test_settings_as_given(checkpoint):
    assert built(checkpoint)[1:4] == (10, 1.0, 1.0)
    assert built(checkpoint, "teacher_k=null", "teacher_weight=null")[1:4] == (10, 1.0, 1.0)
    assert built(checkpoint, "teacher_k=5", "teacher_temperature=2.0", "teacher_weight=0.5")[1:4] == (5, 2.0, 0.5)


def test_numbers_that_the_command_line_reads_as_text(checkpoint):
    assert built(checkpoint, "teacher_weight=1e-3", "teacher_temperature=1e1")[2:4] == (10.0, 0.001)     # (YAML wants a point)


@pytest.mark.parametrize("zero", ["0", "0.0"])
def test_a_weight_of_zero_is_zero(checkpoint, zero):
    assert built(checkpoint, f"teacher_weight={zero}")[3] == 0.0


@pytest.mark.parametrize("bad", ["teacher_k=0", "teacher_temperature=0", "teacher_temperature=0.0"])
def test_zeros_that_mean_nothing_are_refused(checkpoint, bad):
    with pytest.raises(ValueError):
        built(checkpoint, bad)


@pytest.mark.parametrize("weight", [float("nan"), float("inf"), float("-inf"), -1.0])
def test_weights_that_are_no_weights_are_refused(weight):
    def module():
        return KGEModule("rgcn", "dismult", 8, 8, 8, 2, 5, 2, "cosine", 1e-3, 0.2, "none", 2, "random")
    student = module()
    with pytest.raises(ValueError, match="weight"):
        student.set_teacher(module(), weight=weight)
    assert not student.has_teacher
    student.set_teacher(module(), weight=0)
    assert student.has_teacher


def _module(dim=8):
    return KGEModule("rgcn", "dismult", dim, dim, dim, 2, 5, 2, "cosine", 1e-3, 0.2, "none", 1, "random")


def test_a_teacher_that_comes_after_the_padded_loop_is_refused():
    from biomedkg_amd.sampled import SaintGraphedKge
    loop = SaintGraphedKge.__new__(SaintGraphedKge)
    loop.module = _module()
    loop.module.set_teacher(_module())
    with pytest.raises(ValueError, match="teacher"):
        loop.step()


@pytest.mark.gpu
def test_padded_loop_around_a_teacher():
    from biomedkg_amd.sampled import SaintGraphedKge
    gen = torch.Generator().manual_seed(1)
    student = _module(32).cuda().train()
    loop = SaintGraphedKge(student, torch.randn(300, 32, generator=gen).cuda(), torch.randint(0, 300, (2, 2500), generator=gen).cuda(),
                           torch.randint(0, 5, (2500,), generator=gen).cuda(), 8, 4, None)
    assert bool(torch.isfinite(loop.step()))
    student.set_teacher(_module(32))
    with pytest.raises(ValueError, match="teacher"):
        loop.step()
    student.set_teacher(None)
    assert bool(torch.isfinite(loop.step()))
    torch.cuda.synchronize()
    loop.close()


def test_a_module_pickled_before_there_were_teachers_has_none():
    state = _module().__dict__
    state.pop("_teacher", None)                              # (whole-module pickles hold the attributes of their time)
    module = KGEModule.__new__(KGEModule)
    module.__setstate__(state)
    assert not module.has_teacher and module._teacher is None
    module.set_teacher(_module())
    assert module.has_teacher
