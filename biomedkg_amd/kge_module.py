"""KGE task module behind the reference's ``biomedkg/kge_module.py`` API (same constructor kwargs --
all required, no defaults -- hooks, properties and attribute tree).  The arithmetic is
the HIP path: fused modality projection -> R-GCN -> device negative sampling -> DistMult / TransE
scorer -> BCE-with-logits + 1e-2 L2 regulariser.
"""
from __future__ import annotations

from typing import Tuple

import torch
import torch.nn.functional as F

from . import rand as _rand
from .compat import LightningModule
from .factory import FusionFactory, KGEModelFactory
from .gcl_module import _get_scheduler
from .utils.metrics import AUROC, AveragePrecision, BootStrapper, EdgeWisePrecision, F1Score, MetricCollection

# BKG_GROUPED_NEG_TYPES=1: the negatives' relation ids grouped by relation instead of shuffled (ops.grouped_types: the same
# distribution of typed negatives, no permutation launch and no relation sort per step).  The default (round 6) is the
# reference's literal ``edge_type.repeat(k)[randperm]``: the one-pass walk of the negatives needs no relation order, so the
# literal form costs a whole-graph bf16 step 0.08 ms (it cost the two-pass scorer 0.35 ms: rounds 3-5 defaulted to grouping)
GROUPED_NEG_TYPES = __import__("os").environ.get("BKG_GROUPED_NEG_TYPES", "0") == "1"


class KGEModule(LightningModule):
    _teacher = None      # (of the class: a module that was pickled before there were teachers has none)

    def __init__(self, encoder_name: str, decoder_name: str, in_dim: int, hidden_dim: int, out_dim: int,
                 num_hidden_layers: int, num_relation: int, num_heads: int, scheduler_type: str, learning_rate: float,
                 warm_up_ratio: float, fuse_method: str, neg_ratio: int, node_init_method: str):
        super().__init__()
        self.save_hyperparameters()
        self.modality_transform = (FusionFactory.create_fuser(method=fuse_method, embed_dim=in_dim)
                                   if node_init_method == "lm" else None)
        self.model = KGEModelFactory.get_model(
            encoder_name=encoder_name, decoder_name=decoder_name, in_dim=in_dim, hidden_dim=hidden_dim,
            out_dim=out_dim, num_hidden_layers=num_hidden_layers, num_relation=num_relation, num_heads=num_heads)
        self.lr, self.scheduler_type, self.warm_up_ratio, self.neg_ratio = (learning_rate, scheduler_type,
                                                                            warm_up_ratio, neg_ratio)
        metrics = MetricCollection({
            "AUROC": BootStrapper(AUROC(task="binary")),
            "AveragePrecision": BootStrapper(AveragePrecision(task="binary")),
            "F1": BootStrapper(F1Score(task="binary")),
        })
        self._edge_index_map = dict()
        self.valid_metrics = metrics.clone(prefix="val_")
        self.test_metrics = metrics.clone(prefix="test_")
        self._fix_edge_id = None

    def fusion_fn(self, x) -> torch.Tensor:
        """reference kge_module.py:77-84."""
        if self.modality_transform:
            x = self.modality_transform(x)
        elif x.dim() == 3:
            x = torch.mean(x, dim=1)
        return x

    def sample_neg_edges(self, edge_index: torch.Tensor, edge_type: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """reference kge_module.py:86-102: uniform non-edges; relation ids = a random permutation of
        the positives' ids repeated ``neg_ratio`` times."""
        r = _rand.current()
        num_neg_samples = self.neg_ratio * edge_index.size(-1) if self.neg_ratio else None
        neg_edge_index = r.neg_edges(edge_index, num_neg_samples)
        if self.neg_ratio:
            neg_edge_type = None
            rel = getattr(getattr(self.model, "decoder", None), "rel_emb", None)
            if (GROUPED_NEG_TYPES and rel is not None and hasattr(r, "grouped_types")
                    and getattr(neg_edge_index, "_bkg_exchangeable", False)
                    and neg_edge_index.size(1) == num_neg_samples):
                # device randomness: the same multiset of ids in relation order -- a uniformly random pairing all the same,
                # BECAUSE the negatives come out of the keyed-permutation sampler in exchangeable order (the sampler says
                # so on the tensor).  The dense fallback of tiny / dense batches enumerates the population in (head, tail)
                # order: there the ids are shuffled, as the reference does
                neg_edge_type = r.grouped_types(edge_type, self.neg_ratio, rel.size(0))
            if neg_edge_type is None:                                         # == repeat(..)[randperm(..)]
                neg_edge_type = (r.shuffle_repeat(edge_type, self.neg_ratio) if hasattr(r, "shuffle_repeat")
                                 else r.shuffle(edge_type.repeat(self.neg_ratio)))
        else:
            neg_edge_type = edge_type
        return neg_edge_index, neg_edge_type

    def forward(self, x, edge_index, edge_type):
        x = self.fusion_fn(x=x)
        return self.model.encode(x, edge_index, edge_type)

    def _score_step(self, batch):
        """Shared body of the three steps (reference kge_module.py:110-125, 135-150, 175-190)."""
        x = self.fusion_fn(x=batch.x)
        if self._fix_edge_id is not None:
            batch.edge_type = torch.full_like(batch.edge_type, self._fix_edge_id)
        z = self.model.encode(x, batch.edge_index, batch.edge_type)
        neg_edge_index, neg_edge_type = self.sample_neg_edges(batch.edge_index, batch.edge_type)
        pos_pred = self.model.decode(z, batch.edge_index, batch.edge_type)
        neg_pred = self.model.decode(z, neg_edge_index, neg_edge_type)
        pred = torch.cat([pos_pred, neg_pred])
        gt = torch.cat([torch.ones_like(pos_pred), torch.zeros_like(neg_pred)])
        return z, pos_pred, neg_pred, pred, gt

    def _loss(self, z, pred, gt):
        """reference kge_module.py:127-129."""
        cross_entropy_loss = F.binary_cross_entropy_with_logits(pred, gt)
        reg_loss = z.pow(2).mean() + self.model.decoder.rel_emb.pow(2).mean()
        return cross_entropy_loss + 1e-2 * reg_loss

    def _fused_training_loss(self, batch):
        """training_step's arithmetic (reference kge_module.py:110-129) with decode(pos) + decode(neg) + BCE
        fused into one op (``ops.kge_bce_loss``); same loss value and gradients as ``_score_step`` + ``_loss``."""
        from . import ops
        x = self.fusion_fn(x=batch.x)
        if self._fix_edge_id is not None:
            batch.edge_type = torch.full_like(batch.edge_type, self._fix_edge_id)
        z = self.model.encode(x, batch.edge_index, batch.edge_type)
        neg_edge_index, neg_edge_type = self.sample_neg_edges(batch.edge_index, batch.edge_type)
        dec = self.model.decoder
        loss, pos_pred, neg_pred, inverse = ops.kge_bce_loss(z, dec.rel_emb, batch.edge_index, batch.edge_type, neg_edge_index,
                                                             neg_edge_type, dec.kind, reg=1e-2,      # BCE + 1e-2 (mean z^2 + mean rel^2)
                                                             lazy_scores=True)
        if self._teacher is not None and batch.edge_index.size(1) > 0:
            loss = loss + self._distillation_term(batch, z)
        # (detached: must not keep the step's autograd graph alive; the positives' scores may still be in the order of the
        # scorer's sorted frame: ``_last_scores`` puts them in the batch's order when somebody reads them)
        self._scores_of_last_step = (z.detach(), pos_pred, neg_pred, inverse)
        return loss

    @property
    def _last_scores(self):
        """``(z, pos_pred, neg_pred)`` of the last fused training step, the predictions in the batch's triplet order."""
        from . import ops
        last = getattr(self, "_scores_of_last_step", None)
        if last is None:
            return None                              # no fused training step has run yet
        z, pos_pred, neg_pred, inverse = last
        if inverse is not None or isinstance(neg_pred, ops.LazyScores):
            if inverse is not None:
                pos_pred = ops.scores_in_order(pos_pred, inverse)
            if isinstance(neg_pred, ops.LazyScores):      # (the negatives' one-pass walk writes no scores: computed on demand)
                neg_pred = neg_pred()
            self._scores_of_last_step = (z, pos_pred, neg_pred, None)
        return z, pos_pred, neg_pred


    # ------------------------------------------------------------------ entity prediction (no counterpart in the reference)
    def set_teacher(self, teacher, k=10, temperature=1.0, weight=1.0, queries=128):
        """Distil from ``teacher`` (another :class:`KGEModule` over the same nodes and relations, any width): every training
        step adds ``weight`` times the distillation loss of ``queries`` random edges of its batch, each predicting its tail and its
        head out of ALL entities of the batch, against the teacher's ``k`` best entities (:func:`ops.topk_distill_loss`).
        ``None`` switches it off; a ``weight`` of 0 keeps the term and adds nothing.  The teacher is frozen and is no part of this
        module's parameters or state."""
        if teacher is None:
            self._teacher = None
            return
        for m, who in ((self, "student"), (teacher, "teacher")):
            if not hasattr(m.model.decoder, "entity_logits"):
                raise NotImplementedError(f"distillation over entities is implemented for DistMult decoders (the {who}'s is "
                                          f"{type(m.model.decoder).__name__})")
        temperature, weight = float(temperature), float(weight)
        if not (1 <= k <= 1024 and 1e-18 <= temperature <= 1e18 and queries >= 1):
            raise ValueError("set_teacher: k between 1 and 1024, the temperature between 1e-18 and 1e18, at least one query")
        if not 0.0 <= weight < float("inf"):
            raise ValueError(f"set_teacher: the weight must be finite and not negative, got {weight}")
        if teacher is self:
            raise ValueError("set_teacher: a module is not its own teacher (it would be frozen)")
        if teacher.model.decoder.rel_emb.size(0) != self.model.decoder.rel_emb.size(0):
            raise ValueError(f"set_teacher: the teacher knows {teacher.model.decoder.rel_emb.size(0)} relations, the student "
                             f"{self.model.decoder.rel_emb.size(0)}")
        teacher.eval().requires_grad_(False)
        self._teacher = (teacher, int(k), temperature, weight, int(queries))     # (a tuple: not a submodule)

    @property
    def has_teacher(self):
        return self._teacher is not None

    def distillation_loss(self, z, anchor, relation, teacher_ids, teacher_logits, temperature=1.0):
        """Mean over the queries ``(anchor, relation)`` of the distillation loss against a teacher's best entities
        ``teacher_ids / teacher_logits [B, K]`` (id -1: no entry); gradients flow into ``z`` and the relation rows."""
        from . import ops
        return ops.topk_distill_loss(self.model.decoder.entity_logits(z, anchor, relation), teacher_ids, teacher_logits,
                                     temperature)

    @torch.no_grad()
    def top_entities(self, z, anchor, relation, k, table=None):
        """The ``k`` best entities of each query and their scores, ``([B, k] int64, [B, k] fp32)``.  ``table``:
        ``ops.mx4_quantize(z)``, made once per set of embeddings -- the queries are then scored against the 4-bit table (an
        eighth of the bytes of ``z``; its rounding moves scores by a few percent)."""
        best = torch.topk(self.model.decoder.entity_logits(z, anchor, relation, table=table), min(int(k), z.size(0)), dim=1)
        return best.indices, best.values

    def _distillation_term(self, batch, z):
        teacher, k, temperature, weight, queries = self._teacher
        e = torch.randint(0, batch.edge_index.size(1), (queries,), device=z.device)
        relation = batch.edge_type[e].repeat(2)
        anchor = batch.edge_index[:, e].reshape(-1)                  # heads (their tails are asked for), then tails
        with torch.no_grad():
            if next(teacher.parameters()).device != z.device:
                teacher.to(z.device)
            zt = teacher(batch.x, batch.edge_index, batch.edge_type)
            ids, logits = teacher.top_entities(zt, anchor, relation, k)
        return weight * self.distillation_loss(z, anchor, relation, ids, logits, temperature)

    def training_step(self, batch, batch_idx=None):
        if getattr(self.model.decoder, "kind", None) is not None:
            loss = self._fused_training_loss(batch)
        else:
            z, _, _, pred, gt = self._score_step(batch)
            loss = self._loss(z, pred, gt)
        self.log("train_loss", loss, on_epoch=True, on_step=True, prog_bar=True)
        return loss

    def validation_step(self, batch, batch_idx):
        z, pos_pred, _, pred, gt = self._score_step(batch)
        self.valid_metrics.update(pred, gt.to(torch.int32))
        if hasattr(self, "edge_wise_pre_valid"):
            self.edge_wise_pre_valid.update(pos_pred, batch.edge_type)
        loss = self._loss(z, pred, gt)
        self.log("val_loss", loss, on_epoch=True, on_step=True, prog_bar=True)
        return loss

    def on_validation_epoch_end(self):
        output = self.valid_metrics.compute()
        if hasattr(self, "edge_wise_pre_valid"):
            self.log_dict(self.edge_wise_pre_valid.compute())
            self.edge_wise_pre_valid.reset()
        self.log_dict(output)
        self.valid_metrics.reset()

    def test_step(self, batch, batch_idx):
        _, pos_pred, _, pred, gt = self._score_step(batch)
        self.test_metrics.update(pred, gt.to(torch.int32))
        if hasattr(self, "edge_wise_pre_test"):
            self.edge_wise_pre_test.update(pos_pred, batch.edge_type)

    def on_test_epoch_end(self):
        output = self.test_metrics.compute()
        if hasattr(self, "edge_wise_pre_test"):
            self.log_dict(self.edge_wise_pre_test.compute())
            self.edge_wise_pre_test.reset()
        self.log_dict(output)
        self.test_metrics.reset()
        return output

    def configure_optimizers(self):
        params = list(self.model.parameters())
        # torch's fused (single-kernel) Adam on the GPU: the same update as the reference's torch.optim.Adam
        optimizer = torch.optim.Adam(params, lr=self.lr, fused=all(p.is_cuda for p in params) and len(params) > 0)
        return {"optimizer": optimizer, "lr_scheduler": self._get_scheduler(optimizer=optimizer)}

    def _get_scheduler(self, optimizer):
        return _get_scheduler(self, optimizer)

    @torch.no_grad()
    def link_prediction_metrics(self, batch, eval_edge_index=None, eval_edge_type=None, known=None, ks=(1, 3, 10)):
        """Filtered MRR / Hits@k of the DistMult / TransE decoder over ``eval_edge_*`` (default: the batch's own edges),
        embeddings from the batch's message-passing graph.  Not in the reference (it has no ranking metric,
        SURVEY.md 0.2); provided because BASELINE.json's north_star quotes MRR / Hits@k (``biomedkg_amd/eval.py``)."""
        from .eval import distmult_ranking, transe_ranking
        kind = getattr(self.model.decoder, "kind", None)
        if kind not in (0, 1):
            raise NotImplementedError("ranking evaluation is implemented for the DistMult and TransE decoders")
        rank_fn = distmult_ranking if kind == 0 else transe_ranking
        was_training = self.training
        self.eval()
        z = self(batch.x, batch.edge_index, batch.edge_type)
        self.train(was_training)
        ei = batch.edge_index if eval_edge_index is None else eval_edge_index
        et = batch.edge_type if eval_edge_type is None else eval_edge_type
        return rank_fn(z, self.model.decoder.rel_emb, ei, et, known=known, ks=ks)

    @property
    def edge_mapping(self):
        return self._edge_index_map

    @edge_mapping.setter
    def edge_mapping(self, edge_mapping_dict: dict):
        self._edge_index_map = edge_mapping_dict
        self.edge_wise_pre_valid = EdgeWisePrecision(class_mapping=self._edge_index_map)
        self.edge_wise_pre_test = EdgeWisePrecision(class_mapping=self._edge_index_map)

    @property
    def fix_edge_id(self):
        return self._fix_edge_id

    @fix_edge_id.setter
    def fix_edge_id(self, edge_id: int):
        self._fix_edge_id = edge_id
