"""Operators of entity prediction -- one query scored against EVERY entity of the graph (the reference only scores sampled
triplets, ``biomedkg/kge_module.py:109-132``): the scaled lookup of table rows with its gradient by sorted ids, the
distillation loss over the entity logits, and the microscaled 4-bit table a model is served from.  Public names are
re-exported by :mod:`biomedkg_amd.ops`; like everything there they need HIP tensors and launch on torch's current stream.

All of them can be captured into a graph, backward passes included.  As for every operator under autograd, no eager graph over
the same leaf tensors may be alive then (a kept loss of a warm-up step): its accumulation nodes belong to the stream they were
made on, and the capture would be joined with it.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ID_I32 = {torch.int64: False, torch.int32: True}


def _type_of(t, what):
    code = _TYPE.get(t.dtype)
    if code is None:
        raise TypeError(f"{what}: expected float32, bfloat16 or float16, got {t.dtype}")
    return code


def _rows(t):
    """``t`` with its columns next to each other (any row stride; expanded rows are copied out)."""
    return t if (t.stride(1) == 1 or t.size(1) == 1) and (t.stride(0) >= t.size(1) or t.size(0) <= 1) else t.contiguous()


def _ids(t, what):
    if t.dtype not in _ID_I32:
        raise TypeError(f"{what}: expected int64 or int32, got {t.dtype}")


def _on_current_device(what, dev, *others):
    """Everything on one device, the current one: the library launches on its current stream."""
    ok = dev.type == "cuda" and dev.index == L._get_device()
    for t in others:
        ok = ok and (t is None or t.device == dev)
    if not ok:
        _refuse_devices(what, dev, others)


def _refuse_devices(what, dev, others):
    for d in (dev, *(t.device for t in others if t is not None)):
        if d.type != "cuda":
            raise L.HipLibraryError(f"{what}: biomedkg_amd runs on MI355X only: got a tensor on {d} (there is no CPU fallback)")
        if d != dev:
            raise ValueError(f"{what}: tensors on {dev} and {d}")
    raise ValueError(f"{what}: tensors on {dev}, but the current device is cuda:{L._get_device()} (use torch.cuda.device)")


def _refuse_tangents(what, *tensors):
    """Forward-mode derivatives are not implemented: an input that carries one is refused, whether or not a gradient is recorded
    (an autograd function refuses it by itself, but a call that records nothing does not go through one).  Callers look at the
    current level first: outside every ``dual_level`` no tensor carries one."""
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{what}: forward-mode derivatives are not implemented")


# ----------------------------------------------------------------------------- embedding
def _embed_rows(weight, ids, scale):
    w = weight if weight.is_contiguous() else _rows(weight)
    v, d = w.shape
    out = w.new_empty(ids.shape + (d,))
    rc = L.lib().bkg_embed_rows(w.data_ptr(), _TYPE[w.dtype], w.stride(0), v, d, ids.data_ptr(), _ID_I32[ids.dtype], ids.numel(),
                                scale, out.data_ptr(), d, L.stream())
    if rc:
        L.failed("bkg_embed_rows", rc)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, pad):
        out = _embed_rows(weight, ids, scale)
        ctx.save_for_backward(ids)
        v, d = weight.shape
        n = ids.numel()
        lib = L.lib()
        # (what the backward's call takes beside tensors, made here: autograd's thread starts with cold caches, every lookup there
        # counts twice.  Addresses are taken there: hooks may have moved what was saved)
        ctx.call = (lib.bkg_embed_grad, _TYPE[weight.dtype], v, d, n, lib.bkg_embed_grad_workspace_bytes(n, d),
                    _ID_I32[ids.dtype], pad, scale)
        return out

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():      # (the plain path is once_differentiable's without its wrapping)
            return _embedding_backward_once(ctx, g)
        (ids,) = ctx.saved_tensors
        grad, code, v, d, n, ws_bytes, ids_i32, pad, scale = ctx.call
        if g.dim() != 2 or g.stride() != (d, 1):
            g = _rows(g.reshape(n, d))
        dw = g.new_empty((v, d))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=g.device) if ws_bytes else None
        rc = grad(g.data_ptr(), code, g.stride(0), d, ids.data_ptr(), ids_i32, n, v, pad, scale, dw.data_ptr(),
                  ws.data_ptr() if ws_bytes else None, ws_bytes, L.stream())
        if rc:
            L.failed("bkg_embed_grad", rc)
        return dw, None, None, None


_embedding_backward_once = once_differentiable(lambda ctx, g: _Embedding.backward(ctx, g))


def _check_embedding(weight, ids):
    if weight.dim() != 2:
        raise ValueError(f"embedding: expected a [V, d] table, got {tuple(weight.shape)}")
    _type_of(weight, "embedding")
    if _forward_ad._current_level >= 0:
        _refuse_tangents("embedding", weight)
    _ids(ids, "embedding ids")
    _on_current_device("embedding", weight.device, ids)


def embedding(weight, ids, scale=1.0, padding_idx=None):
    """``scale * weight[ids]`` -> ``ids.shape + (d,)`` in ``weight``'s type (fp32 / bf16 / fp16, one rounding).

    ``weight [V, d]`` (any row stride), ``ids`` int64 / int32 of any shape.  An id outside ``[0, V)`` reads as a row of zeros
    and gets no gradient (padded batches); ``padding_idx`` (negative: from the end) reads its row and gets no gradient.

    The gradient is dense ``[V, d]`` in ``weight``'s type: ids sorted (stable), every row summed in fp32 in the order of its
    positions, rounded once -- bitwise repeatable, no atomics (csrc/embed.hip)."""
    _check_embedding(weight, ids)
    v, d = weight.shape
    if v >= 2 ** 31 or ids.numel() >= 2 ** 31 or d > 2 ** 20:
        raise ValueError("embedding: at most 2^31 - 1 rows and ids, 2^20 columns")
    scale = float(scale)
    pad = -1
    if padding_idx is not None:
        if not -v <= padding_idx < v:
            raise ValueError(f"embedding: padding_idx {padding_idx} outside the table's {v} rows")
        pad = int(padding_idx) % v
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(weight, ids, scale, pad)
    return _embed_rows(weight, ids, scale)


# ----------------------------------------------------------------------------- distillation
def _distill_forward(x, ids, t, temp, sum_scale, want_sum, d=None):
    rows, v = x.shape
    dev, xt = x.device, _TYPE[x.dtype]
    lib = L.lib()
    # one buffer: the row statistics (kept for the backward), the rows' losses, the launches' scratch
    n_ws = lib.bkg_distill_workspace_floats(rows, v, xt)
    stats = torch.empty(4 * rows + (rows if want_sum else 0) + n_ws, dtype=torch.float32, device=dev)
    out = torch.empty(() if want_sum else (rows,), dtype=torch.float32, device=dev)
    base, to = stats.data_ptr(), out.data_ptr()
    losses, scratch = (base + 16 * rows, base + 20 * rows) if want_sum else (to, base + 16 * rows)
    rc = lib.bkg_distill_forward(x.data_ptr(), xt, x.stride(0), rows, v, ids.data_ptr(), _ID_I32[ids.dtype], ids.stride(0),
                                 t.data_ptr(), _TYPE[t.dtype], t.stride(0), ids.size(1), temp, sum_scale, scratch, base, losses,
                                 to if want_sum else None, None if d is None else d.data_ptr(), v, L.stream())
    if rc:
        L.failed("bkg_distill_forward", rc)
    return out, stats


class _TopkDistill(torch.autograd.Function):
    """A reduced loss leaves its gradient (for an upstream factor of 1) with the forward, while the logits lie in the caches;
    the first backward hands it out -- the launch there looks at the factor on the device and computes the gradient again
    where it is not 1.  A later backward over the same graph, a captured one, and reduction "none" compute it afresh."""

    @staticmethod
    def forward(ctx, x, ids, t, temp, mean, want_sum):
        sum_scale = 1.0 / x.size(0) if mean else 1.0
        d = None
        if want_sum and not torch.cuda.is_current_stream_capturing():
            d = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        out, stats = _distill_forward(x, ids, t, temp, sum_scale, want_sum, d)
        ctx.save_for_backward(x, ids, t, stats)
        ctx.made = d
        # (as for the lookup: what the backward's call takes beside tensors, made here)
        ctx.call = (L.lib().bkg_distill_backward, _TYPE[x.dtype], _ID_I32[ids.dtype], _TYPE[t.dtype], ids.size(1), temp,
                    int(not want_sum), temp * sum_scale)
        return out

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            # (the gradient depends on the logits too: a second derivative is refused even where g itself records none)
            return _distill_backward_once(ctx, g if g.requires_grad else g.detach().requires_grad_())
        x, ids, t, stats = ctx.saved_tensors
        d, ctx.made = ctx.made, None
        grad, xt, ids_i32, tt, k, temp, g_step, coef = ctx.call
        rows, v = x.shape
        kept = d is not None and not torch.cuda.is_current_stream_capturing()
        if not kept:
            d = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        if g.dtype != torch.float32 or not g.is_contiguous():
            g = g.to(torch.float32).contiguous()
        rc = grad(x.data_ptr(), xt, x.stride(0), rows, v, ids.data_ptr(), ids_i32, ids.stride(0), t.data_ptr(), tt, t.stride(0),
                  k, temp, stats.data_ptr(), g.data_ptr(), g_step, coef, kept, d.data_ptr(), v, L.stream())
        if rc:
            L.failed("bkg_distill_backward", rc)
        return d, None, None, None, None, None


_distill_backward_once = once_differentiable(lambda ctx, g: _TopkDistill.backward(ctx, g))


def topk_distill_loss(logits, teacher_ids, teacher_logits, temperature=1.0, reduction="batchmean"):
    """Distillation of ``logits [R, V]`` (fp32 / bf16 / fp16) from a teacher's best entries: ``teacher_ids [R, K]`` (int64 /
    int32) with ``teacher_logits [R, K]`` (constants: no gradient flows into them), ``1 <= K <= 1024``.

    Per row ``T^2 * KL(q || p)`` over the K entries with ``q = softmax(teacher_logits / T)`` over the row's usable entries and
    ``p = softmax(logits / T)`` over all V columns; the gradient is ``T * (p - q)`` in ``logits``'s type, statistics and sums in
    fp32 (csrc/distill.hip).  ``K = 1`` is cross entropy.  A reduced loss that records gradients computes its gradient within
    the forward call (one pass over the logits less; the backward repeats it only for an upstream factor other than 1).  An entry is not usable if its id lies outside ``[0, V)`` (padding:
    -1) or its logit is ``-inf``; an id that occurs twice counts twice.  A row without a usable entry, or whose logits are all
    ``-inf``, is left out: loss 0, gradient 0.  A usable entry whose student logit is ``-inf`` makes the loss ``inf``; NaN stays
    NaN.

    ``reduction``: ``"batchmean"`` (sum / R), ``"sum"`` -> fp32 scalars, ``"none"`` -> fp32 ``[R]``."""
    if logits.dim() != 2 or teacher_ids.dim() != 2 or teacher_logits.shape != teacher_ids.shape \
            or teacher_ids.size(0) != logits.size(0):
        raise ValueError(f"topk_distill_loss: expected logits [R, V] and teacher ids / logits [R, K], got {tuple(logits.shape)}, "
                         f"{tuple(teacher_ids.shape)}, {tuple(teacher_logits.shape)}")
    _type_of(logits, "topk_distill_loss logits")
    _type_of(teacher_logits, "topk_distill_loss teacher logits")
    _ids(teacher_ids, "topk_distill_loss teacher ids")
    if _forward_ad._current_level >= 0:
        _refuse_tangents("topk_distill_loss", logits, teacher_logits)
    _on_current_device("topk_distill_loss", logits.device, teacher_ids, teacher_logits)
    if reduction not in ("batchmean", "sum", "none"):
        raise ValueError(f"topk_distill_loss: reduction {reduction!r} (batchmean, sum or none)")
    temp = float(temperature)
    if not 1e-18 <= temp <= 1e18:
        raise ValueError(f"topk_distill_loss: the temperature must lie between 1e-18 and 1e18, got {temperature}")
    rows, v = logits.shape
    k = teacher_ids.size(1)
    if not 1 <= k <= 1024:
        raise ValueError(f"topk_distill_loss: between 1 and 1024 teacher entries per row, got {k}")
    if v == 0 or v >= 2 ** 30 or rows >= 2 ** 22:
        raise ValueError("topk_distill_loss: between 1 and 2^30 - 1 columns, below 2^22 rows")
    if teacher_logits.requires_grad:
        raise ValueError("topk_distill_loss: the teacher's logits are constants (detach them)")
    if rows == 0:
        z = logits.float().sum(1)
        return z if reduction == "none" else z.sum()
    ids, t = _rows(teacher_ids), _rows(teacher_logits)
    want_sum = reduction != "none"
    mean = reduction == "batchmean"
    if logits.requires_grad and torch.is_grad_enabled():
        return _TopkDistill.apply(_rows(logits), ids, t, temp, mean, want_sum)
    return _distill_forward(_rows(logits), ids, t, temp, 1.0 / rows if mean else 1.0, want_sum)[0]


# ----------------------------------------------------------------------------- microscaled 4-bit tables
class Mx4Table:
    """A ``[rows, cols]`` table in microscaled 4 bits (:func:`mx4_quantize`), in panels of 128 columns (the last one padded
    with zeros): ``codes`` uint8 ``[panels, rows, 64]`` (two columns a byte, the lower one in the low nibble) and ``scales``
    uint8 ``[panels, rows, 4]`` (the exponent of each 32 columns + 127; 255: the block held an infinity or NaN).  0.53 bytes a
    value.  May be copied, pickled and saved; made of given parts, their memory has to stay where it is."""
    __slots__ = ("shape", "device", "codes_ptr", "scales_ptr", "_store")

    def __init__(self, codes, scales, shape):
        rows, cols = shape
        panels = (cols + 127) // 128
        for t, want, what in ((codes, (panels, rows, 64), "codes"), (scales, (panels, rows, 4), "scales")):
            if t.dtype != torch.uint8 or tuple(t.shape) != want or not t.is_contiguous():
                raise ValueError(f"Mx4Table: {what} must be contiguous uint8 {want} for a table of {tuple(shape)}")
        if codes.device != scales.device:
            raise ValueError(f"Mx4Table: codes on {codes.device}, scales on {scales.device}")
        if codes.data_ptr() % 16 or scales.data_ptr() % 4:
            raise ValueError("Mx4Table: codes must be 16-byte, scales 4-byte aligned")
        self.shape, self.device = (rows, cols), codes.device
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()
        self._store = (codes, scales)

    @classmethod
    def _of(cls, store, rows, cols):
        """A table in one piece of memory: the codes, then the scales."""
        self = cls.__new__(cls)
        self.shape, self.device = (rows, cols), store.device
        self.codes_ptr = store.data_ptr()
        self.scales_ptr = self.codes_ptr + (cols + 127) // 128 * rows * 64
        self._store = store
        return self

    @classmethod
    def _empty(cls, rows, cols, device):
        return cls._of(torch.empty((cols + 127) // 128 * rows * 68, dtype=torch.uint8, device=device), rows, cols)

    def __reduce__(self):
        """Copies and saved tables (``copy``, ``pickle``, ``torch.save``) are made from the memory and the shape: device and
        addresses are those of the copy's own memory."""
        if self._store.__class__ is tuple:
            return Mx4Table, (*self._store, self.shape)
        return _table_in_one_piece, (self._store, self.shape)

    def __setstate__(self, state):
        """A table that was saved with its attributes: only its memory and shape are taken, its addresses are another process's."""
        _, saved = state
        store, (rows, cols) = saved["_store"], saved["shape"]
        if store.__class__ is tuple:
            table = Mx4Table(*store, (rows, cols))
        else:
            table = _table_in_one_piece(store, (rows, cols))
        for name in self.__slots__:
            setattr(self, name, getattr(table, name))

    def _parts(self):
        store = self._store
        if store.__class__ is tuple:
            return store
        rows, panels = self.shape[0], (self.shape[1] + 127) // 128
        cut = panels * rows * 64
        return store[:cut].view(panels, rows, 64), store[cut:].view(panels, rows, 4)

    @property
    def codes(self):
        return self._parts()[0]

    @property
    def scales(self):
        return self._parts()[1]

    @property
    def nbytes(self):
        return (self.shape[1] + 127) // 128 * self.shape[0] * 68

    def __repr__(self):
        return f"Mx4Table({self.shape[0]} x {self.shape[1]}, {self.nbytes} bytes, {self.device})"


def _table_in_one_piece(store, shape):
    rows, cols = shape
    if store.dtype != torch.uint8 or store.shape != ((cols + 127) // 128 * rows * 68,) or not store.is_contiguous() \
            or store.data_ptr() % 16:
        raise ValueError(f"Mx4Table: no packed table of {tuple(shape)}")
    return Mx4Table._of(store, rows, cols)


def mx4_quantize(x):
    """``x [rows, cols]`` (fp32 / bf16 / fp16) as an :class:`Mx4Table`: per 32 columns the shared scale is
    ``2^(floor(log2(max|x|)) - 2)`` (exponent within [-127, 127]), values go to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 times
    it, ties to the even code (csrc/mx4.hip).  No gradient."""
    if x.dim() != 2 or x.size(1) == 0:
        raise ValueError(f"mx4_quantize: expected [rows, cols] with cols > 0, got {tuple(x.shape)}")
    _type_of(x, "mx4_quantize")
    _on_current_device("mx4_quantize", x.device)
    rows, cols = x.shape
    if cols > 2 ** 24 or rows >= 2 ** 31:
        raise ValueError("mx4_quantize: at most 2^24 columns and 2^31 - 1 rows")
    if not x.is_contiguous():
        x = _rows(x.detach())
    table = Mx4Table._empty(rows, cols, x.device)
    rc = L.lib().bkg_mx4_quantize(x.data_ptr(), _TYPE[x.dtype], x.stride(0), rows, cols, table.codes_ptr, table.scales_ptr, L.stream())
    if rc:
        L.failed("bkg_mx4_quantize", rc)
    return table


def mx4_dequantize(table, dtype=torch.float32):
    """The values an :class:`Mx4Table` holds, ``[rows, cols]`` in ``dtype`` (exact in fp32 and bf16; fp16 rounds)."""
    if not isinstance(table, Mx4Table):
        raise TypeError("mx4_dequantize: expected an Mx4Table")
    if dtype not in _TYPE:
        raise TypeError(f"mx4_dequantize: float32, bfloat16 or float16, got {dtype}")
    _on_current_device("mx4_dequantize", table.device)
    rows, cols = table.shape
    out = torch.empty(rows, cols, dtype=dtype, device=table.device)
    rc = L.lib().bkg_mx4_dequantize(table.codes_ptr, table.scales_ptr, rows, cols, out.data_ptr(), _TYPE[dtype], cols, L.stream())
    if rc:
        L.failed("bkg_mx4_dequantize", rc)
    return out


def mx4_linear(x, table, bias=None, out_dtype=None):
    """``x @ table.T (+ bias)`` with both operands in microscaled 4 bits, products and sums on the matrix cores in fp32, one
    rounding into ``out_dtype`` (default: ``x``'s type).  ``x [..., cols]`` fp32 / bf16 / fp16 is quantised within the call
    (or is an :class:`Mx4Table` already: then ``out_dtype`` defaults to fp32), ``table [n, cols]``, ``bias [n]`` fp32.

    For inference: no gradient (an input that requires one is refused while gradients are recorded)."""
    if not isinstance(table, Mx4Table):
        raise TypeError("mx4_linear: the table must be an Mx4Table (mx4_quantize)")
    n, cols = table.shape
    if bias is not None and (bias.shape != (n,) or bias.dtype != torch.float32 or not bias.is_contiguous()):
        raise ValueError(f"mx4_linear: bias must be contiguous fp32 [{n}]")
    packed = isinstance(x, Mx4Table)
    if ((bias is not None and bias.requires_grad) or (not packed and x.requires_grad)) and torch.is_grad_enabled():
        raise ValueError("mx4_linear is an inference product without a gradient (call it under torch.no_grad())")
    if (x.shape[-1] if len(x.shape) else -1) != cols:
        raise ValueError(f"mx4_linear: x {tuple(x.shape)} against a table of {cols} columns")
    out_dtype = out_dtype or (torch.float32 if packed else x.dtype)
    if out_dtype not in _TYPE:
        raise TypeError(f"mx4_linear: out_dtype float32, bfloat16 or float16, got {out_dtype}")
    if packed:
        if _forward_ad._current_level >= 0:
            _refuse_tangents("mx4_linear", bias)
        _on_current_device("mx4_linear", table.device, x, bias)
        m = x.shape[0]
        out = torch.empty(m, n, dtype=out_dtype, device=table.device)
        ws_bytes = L.lib().bkg_mx4_matmul_workspace_bytes(m, n, cols)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=table.device) if ws_bytes else None
        L.call("bkg_mx4_matmul", x.codes_ptr, x.scales_ptr, m, table.codes_ptr, table.scales_ptr, n, cols, L.ptr(bias),
               out.data_ptr(), _TYPE[out_dtype], n, L.ptr(ws), ws_bytes, L.stream())
        return out
    xt = _type_of(x, "mx4_linear")
    if _forward_ad._current_level >= 0:
        _refuse_tangents("mx4_linear", x, bias)
    _on_current_device("mx4_linear", x.device, table, bias)
    lib = L.lib()
    x2 = x if x.dim() == 2 else x.reshape(-1, cols)
    if not x2.is_contiguous():
        x2 = _rows(x2)
    m = x2.size(0)
    out = torch.empty(x.shape[:-1] + (n,), dtype=out_dtype, device=x.device)
    ws_bytes = lib.bkg_mx4_linear_workspace_bytes(m, n, cols)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device) if ws_bytes else None
    rc = lib.bkg_mx4_linear(x2.data_ptr(), xt, x2.stride(0), m, table.codes_ptr, table.scales_ptr, n, cols, L.ptr(bias),
                            out.data_ptr(), _TYPE[out_dtype], n, L.ptr(ws), ws_bytes, L.stream())
    if rc:
        L.failed("bkg_mx4_linear", rc)
    return out
