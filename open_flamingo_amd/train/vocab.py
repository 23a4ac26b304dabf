"""The two ends of a language model on its vocabulary table, for training the whole table: the scaled lookup with a gradient by sorted
tokens and the (tied) head's cross entropy without logits.

Both are plain functions on tensors (``embedding_lookup``, ``linear_cross_entropy``); ``use_libofhip_vocab`` routes a Hugging Face causal LM
through them.  They stand beside ``towers.use_libofhip_lm_loss``, which computes the same loss from materialised logits, and
``sparse_rows``, which trains two rows of a frozen table.  GPU tensors only, like everything that runs on libofhip.
"""
import threading
import types

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ..hip import abi
from ..hip.ops import BF16, F32, Ops
from ..src import helpers
from ..src.utils import extend_instance

_REDUCTION = {"none": abi.CE_NONE, "mean": abi.CE_MEAN, "sum": abi.CE_SUM}


def _rows16(t):
    """``t`` with unit column stride and rows that begin at multiples of 16 bytes (itself where it has them)."""
    per = 16 // t.element_size()
    if t.stride(-1) == 1 and t.stride(0) % per == 0 and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous() if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _elsewhere(t):
    """a context for launches on ``t``'s device, or None where that is the current one (nothing to enter: host time of small calls)"""
    at = t.get_device()
    return None if at < 0 or at == torch.cuda.current_device() else torch.cuda.device(at)


def _forward_mode():
    """Tangents may be attached to the operands (forward-mode AD: inside a dual level, with gradients switched off as well)."""
    return forward_ad._current_level >= 0


def _needs_node(*tensors):
    """The call has to be an autograd node: an operand wants a gradient, or may carry a tangent, which a bare launch would drop and the node
    refuses (NotImplementedError: the operators have a backward only)."""
    return _forward_mode() or (torch.is_grad_enabled() and any(t.requires_grad for t in tensors))


def _backward(run, ctx, g):
    """``run(ctx, g)`` on g's device.  Under create_graph the result is marked as differentiable once; without it there is no graph to mark,
    and the marking's host time (as long as a small call's kernels) is left out."""
    if torch.is_grad_enabled():
        run = once_differentiable(run)
    other = _elsewhere(g)
    if other is None:
        return run(ctx, g)
    with other:
        return run(ctx, g)


def _linear_ce(hidden, table, labels, kw, ops, need):
    """(loss, what a backward needs)"""
    x, w = _rows16(hidden), _rows16(table)
    loss_rows = x.new_empty(x.shape[0], dtype=F32)
    loss = x.new_empty((), dtype=F32) if kw["reduction"] != abi.CE_NONE else None
    state = ops.linear_ce_fwd(x, w, labels, loss_rows, loss, need=need, **kw)
    return loss_rows if loss is None else loss, (x, w, labels, state)


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, table, labels, kw, ops):
        ctx.need = ctx.needs_input_grad[:2]
        loss, saved = _linear_ce(hidden, table, labels, kw, ops, ctx.need)
        ctx.save_for_backward(*saved)
        ctx.kw, ctx.ops = kw, ops
        return loss

    @staticmethod
    def backward(ctx, g):
        return _backward(_LinearCrossEntropy.run_backward, ctx, g)

    @staticmethod
    def run_backward(ctx, g):
        x, w, labels, state = ctx.saved_tensors
        if g.dtype is not F32 or not g.is_contiguous():
            g = g.to(F32).contiguous()
        dx = x.new_empty(x.shape) if ctx.need[0] else None
        dw = w.new_empty(w.shape) if ctx.need[1] else None
        ctx.ops.linear_ce_bwd(x, w, labels, state, g, dx, dw, **ctx.kw)
        return dx, dw, None, None, None


def linear_cross_entropy(hidden, table, labels, *, ignore_index=-100, reduction="mean", logit_scale=1.0, piece=0, ops=None):
    """Softmax cross entropy of the logits ``logit_scale * hidden @ table.T``, which are never stored:
    ``F.cross_entropy(logits.float(), labels, ignore_index=..., reduction=...)`` with fp32 statistics of unrounded logits.

    hidden (..., d) and table (vocabulary, d): bfloat16, or any floating type under bf16 autocast (cast as ``F.linear`` casts); d a
    multiple of 8.  labels (...): int64, already shifted.  reduction "mean" (over the labels that count: NaN without any), "sum" or
    "none" (one fp32 loss per label, 0 where ignored).  A label outside the vocabulary that is not ``ignore_index`` makes the loss NaN and
    has no gradient.

    Gradients come in bfloat16 for both operands, through fp32 sums of products whose one factor, the logits' gradient (softmax - onehot,
    or exp(logit - label's logit) where the table has no gradient), is rounded to bfloat16: half a step, 2^-8 of each entry, on the way.
    Where the table has no gradient the forward prepares the hidden states' one from the same product.  ``piece``: vocabulary rows the
    backward holds a logits gradient of at a time (0: chosen, 128 MB of it).  Differentiable once, backward; forward-mode AD raises."""
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction must be one of {sorted(_REDUCTION)}, got {reduction!r}")
    shape, d, n = hidden.shape, hidden.shape[-1], labels.numel()
    if shape[:-1] != labels.shape:
        raise ValueError(f"labels {tuple(labels.shape)} do not fit hidden states {tuple(shape)}")
    if table.dim() != 2 or table.shape[1] != d or table.shape[0] == 0:
        raise ValueError(f"table {tuple(table.shape)} does not fit hidden states {tuple(shape)}")
    if (n + 255) // 256 * 256 * max((d + 63) // 64 * 64, 256) >= 1 << 31:          # (256 table rows of logits gradient are the least a piece holds)
        raise ValueError(f"{n} rows of {d}: a call must stay below 2^31 elements of hidden states and below 2^23 rows; split the batch")
    if d % 8:
        raise ValueError(f"the hidden size must be a multiple of 8, got {d}")
    if labels.dtype is not torch.int64:
        raise TypeError(f"labels must be int64, got {labels.dtype}")
    if piece < 0:
        raise ValueError("piece must not be negative")
    if not hidden.get_device() == table.get_device() == labels.get_device():
        raise ValueError(f"hidden, table and labels are on {hidden.device}, {table.device} and {labels.device}")
    if ops is None:
        ops = _ops_for(hidden, ops, "linear_cross_entropy")
    if hidden.dtype is not BF16 or table.dtype is not BF16:
        dev = hidden.device.type
        if torch.is_autocast_enabled(dev) and torch.get_autocast_dtype(dev) == BF16:
            hidden, table = hidden.to(BF16), table.to(BF16)
        if hidden.dtype is not BF16 or table.dtype is not BF16:
            raise TypeError(f"linear_cross_entropy takes bfloat16 operands (or runs under bf16 autocast), got {hidden.dtype} and {table.dtype}")
    x = hidden if len(shape) == 2 else hidden.reshape(-1, d)
    y = labels if len(shape) == 2 and labels.is_contiguous() else labels.reshape(-1).contiguous()
    if n == 0:          # no rows: torch's values, zero gradients
        zero = (hidden.sum() + table[:0].sum()).to(F32)
        return zero.expand(labels.shape) if reduction == "none" else zero / 0.0 if reduction == "mean" else zero
    kw = dict(ignore_index=int(ignore_index), logit_scale=float(logit_scale), reduction=_REDUCTION[reduction], piece=int(piece))
    other = _elsewhere(x)
    if other is None:
        out = _run_linear_ce(x, table, y, kw, ops)
    else:
        with other:
            out = _run_linear_ce(x, table, y, kw, ops)
    return out.view(labels.shape) if reduction == "none" and len(shape) != 2 else out


def _run_linear_ce(x, table, y, kw, ops):
    if _needs_node(x, table):
        return _LinearCrossEntropy.apply(x, table, y, kw, ops)
    return _linear_ce(x, table, y, kw, ops, (False, False))[0]


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale, padding_idx, ops):
        out = table.new_empty((ids.shape[0], table.shape[1]))
        ops.embedding_fwd(ids, table, out, scale)
        ctx.save_for_backward(ids)
        ctx.shape, ctx.scale, ctx.padding_idx, ctx.ops = table.shape, scale, padding_idx, ops
        return out

    @staticmethod
    def backward(ctx, g):
        return _backward(_EmbeddingLookup.run_backward, ctx, g)

    @staticmethod
    def run_backward(ctx, g):
        (ids,) = ctx.saved_tensors
        if g.stride(1) != 1 or g.stride(0) < g.shape[1]:
            g = g.contiguous()
        dw = g.new_empty(ctx.shape)
        ctx.ops.embedding_bwd(ids, g, dw, ctx.scale, ctx.padding_idx)
        return None, dw, None, None, None


def _run_embedding(ids, t, scale, padding_idx, ops):
    if _needs_node(t):
        return _EmbeddingLookup.apply(ids, t, scale, padding_idx, ops)
    out = t.new_empty((ids.shape[0], t.shape[1]))
    ops.embedding_fwd(ids, t, out, scale)
    return out


def embedding_lookup(ids, table, *, scale=1.0, padding_idx=None, ops=None):
    """``scale * F.embedding(ids, table, padding_idx)`` for an fp32 or bf16 table, with a dense gradient that is summed in fp32 in a
    fixed order (the same bits on every run) and rounded once.

    ids: int64 of any shape; an id outside the table gives a row of NaN and no gradient.  padding_idx (None: none; negative: counted
    from the table's end): that row gets no gradient.  Differentiable once, backward; forward-mode AD raises."""
    if table.dim() != 2 or 0 in table.shape:
        raise ValueError(f"table must be (vocabulary, d), got {tuple(table.shape)}")
    vocab, d = table.shape
    if ids.dtype is not torch.int64:
        raise TypeError(f"ids must be int64, got {ids.dtype}")
    if table.dtype is not F32 and table.dtype is not BF16:
        raise TypeError(f"the table must be float32 or bfloat16, got {table.dtype}")
    if ids.get_device() != table.get_device():
        raise ValueError(f"ids and table are on {ids.device} and {table.device}")
    if padding_idx is not None:
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"padding_idx {padding_idx} is outside a table of {vocab} rows")
        padding_idx %= vocab
    if ops is None:
        ops = _ops_for(table, ops, "embedding_lookup")
    flat = ids if ids.dim() == 1 and ids.is_contiguous() else ids.reshape(-1).contiguous()
    n = flat.shape[0]
    if n == 0:
        return table[:0].reshape(*ids.shape, d) * scale
    t = table if table.stride(1) == 1 and table.stride(0) >= d else table.contiguous()

    pad = -1 if padding_idx is None else padding_idx
    other = _elsewhere(t)
    if other is None:
        out = _run_embedding(flat, t, float(scale), pad, ops)
    else:
        with other:
            out = _run_embedding(flat, t, float(scale), pad, ops)
    return out if ids.dim() == 1 else out.view(*ids.shape, d)


def _ops_for(t, ops, what):
    """the given Ops (tests: the emulator's), else the product's, which takes GPU tensors only"""
    if ops is not None:
        return ops
    helpers._require_hip(t, what)
    return Ops.default()


# ---------------------------------------------------------------------------------------------------------------- Hugging Face LMs
def _runs_here(t):
    """libofhip takes this table, in plain or reverse-mode execution; everything else (forward-mode AD and torch.func's transforms among it)
    keeps the LM's own modules, which support it"""
    if _forward_mode() or torch._C._are_functorch_transforms_active():
        return False
    try:
        helpers._require_hip(t, "vocabulary table")
    except (RuntimeError, TypeError):
        return False
    return True


def _keeps_all(logits_to_keep):
    return isinstance(logits_to_keep, int) and logits_to_keep == 0


def _plain_product(head):
    """The head is x @ weight.T and nothing besides: no bias, no forward of its own (an adapter's, a patched one), no hooks that would see or change
    the logits."""
    return (isinstance(head, torch.nn.Linear) and type(head).forward is torch.nn.Linear.forward and "forward" not in head.__dict__ and head.bias is None
            and not (head._forward_hooks or head._forward_pre_hooks or head._backward_hooks or head._backward_pre_hooks))


def _embedding_forward(self, ids):
    if ids.dtype == torch.int64 and self.weight.dtype in (F32, BF16) and _runs_here(self.weight):
        return embedding_lookup(ids, self.weight, padding_idx=self.padding_idx)
    return self._of_eager_forward(ids)


class _VocabLossMixin:
    """``forward(labels=...)`` of a Hugging Face causal LM without logits: the output's ``loss`` comes from ``linear_cross_entropy`` on the
    last hidden states and the head's weight, its ``logits`` is None.  Without labels nothing changes.  What the operator does not
    cover (a head with a bias, hooks or a forward of its own, ``logits_to_keep``, other loss arguments, operands that are not bf16 or under bf16 autocast, the two-row mode of
    train/sparse_rows.py, whose tap sits behind the logits) takes the LM's own path."""

    def _of_takes(self, args, kwargs):
        labels = kwargs.get("labels")
        if len(args) > 1:          # (what the second positional argument is differs from LM to LM)
            return False
        head = self.get_output_embeddings()
        w = getattr(head, "weight", None)
        if labels is None or w is None or w.shape[1] % 8 or not _plain_product(head) or not _keeps_all(kwargs.get("logits_to_keep", 0)) or not _runs_here(w):
            return False
        if any(kwargs.get(k) is not None for k in ("num_items_in_batch", "shift_labels", "ignore_index")) or getattr(w, "_of_trained_rows", None) is not None:
            return False
        dev = w.device.type
        return (torch.get_autocast_dtype(dev) if torch.is_autocast_enabled(dev) else w.dtype) == BF16          # what the head would multiply in

    def forward(self, *args, **kwargs):
        if not self._of_takes(args, kwargs):
            return super().forward(*args, **kwargs)
        labels = kwargs.pop("labels")
        kwargs.pop("logits_to_keep", None)
        seen, me = [], threading.get_ident()
        # (the hook sits on a module that other threads may be running as well)
        hook = self.base_model.register_forward_hook(lambda mod, args, out: seen.append(out[0]) if threading.get_ident() == me else None)
        try:          # the LM's own forward with no position for the head: hidden states, cache and all the rest as it makes them
            none = torch.empty(0, dtype=torch.int64, device=labels.device)
            out = super().forward(*args, logits_to_keep=none, **kwargs)
        finally:
            hook.remove()
        w = self.get_output_embeddings().weight
        ahead = torch.nn.functional.pad(labels.to(seen[-1].device), (0, 1), value=-100)[..., 1:]          # position i predicts token i + 1
        loss = linear_cross_entropy(seen[-1], w, ahead.to(torch.int64))
        if isinstance(out, tuple):          # (logits, ...) without labels: (loss, logits, ...) with
            return (loss, None) + out[1:]
        return type(out)(loss=loss, **{k: v for k, v in out.items() if k != "logits"})


def use_libofhip_vocab(lm):
    """Route a Hugging Face causal LM's vocabulary table through libofhip on both ends: the lookup (``embedding_lookup``) and, where labels are
    given, the loss (``linear_cross_entropy``: the output then has no logits).  Before or after the LM becomes part of a Flamingo."""
    known = {"MptForCausalLM", "GPTNeoXForCausalLM"}
    if not known & {c.__name__ for c in type(lm).__mro__}:
        raise NotImplementedError(f"use_libofhip_vocab knows {sorted(known)}, got {type(lm).__name__}")
    if isinstance(lm, _VocabLossMixin):
        return lm
    emb = lm.get_input_embeddings()
    if type(emb) is torch.nn.Embedding and "forward" not in emb.__dict__ and emb.max_norm is None and not emb.scale_grad_by_freq and not emb.sparse:
        emb._of_eager_forward = emb.forward
        emb.forward = types.MethodType(_embedding_forward, emb)
    extend_instance(lm, _VocabLossMixin)
    return lm
