"""Losses over a large vocabulary without keeping the logits, and a teacher's top logits.

  vocab_cross_entropy   softmax cross entropy of hidden states against decoder rows, forward and backward in pieces of the
                        vocabulary (gridmm_vocab_loss_fwd / _bwd).  Beside autograd.linear + torch's cross_entropy, which is what
                        GlocalTextPathCMTPreTraining.forward_mlm (pretrain_src/model/pretrain_cmt.py:131-153) computes and which
                        keeps rows x vocabulary fp32 logits for the backward
  vocab_distillation    the same head against a teacher's top logits: T^2 KL(teacher over its slots || student over everything)
  top_logits            the k largest logits of every row, their ids and the row's log-sum-exp: the teacher's side

There is no CPU fallback: the functions raise on non-GPU tensors.
"""
import contextlib
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib, ops
from .autograd import DEFERRED
from .ops import _p, _stream

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_TOP, MAX_TOP_ROWS = 1024, 1 << 22
MAX_ROWS, MAX_VOCAB, MAX_HIDDEN, MAX_SLOTS = 1 << 20, 1 << 27, 1 << 20, 1 << 16


class _Desc(ctypes.Structure):
    """gridmm_vocab_loss_t of include/gridmm.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("hidden", "weight", "bias", "labels", "ids", "teacher")]
                + [(n, ctypes.c_int64) for n in ("ld_hidden", "ld_weight", "ld_ids", "ld_teacher", "ignore_index")]
                + [(n, ctypes.c_int) for n in ("rows", "vocab", "hidden_size", "slots", "dtype", "bias_dtype", "index64", "forward_only", "packed")]
                + [("temperature", ctypes.c_float)])


_HERE = contextlib.nullcontext()


def _on(device):
    """The tensors' own device as the current one (the kernels go to its current stream)."""
    if device.index == ops._CUR_DEVICE():
        return _HERE
    return torch.cuda.device(device)


def _rows(t):
    """(..., C) -> its rows as (M, C) with a contiguous last dimension and one row stride, and that stride."""
    C = t.shape[-1]
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= C:
        return t, t.stride(0)
    t = t.contiguous().view(-1, C) if C else t.reshape(0, 0)
    return t, C


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _check_head(hidden, weight, bias, *index):
    for t in (hidden, weight, bias) + index:
        if t is None:
            continue
        if not t.is_cuda:
            raise _lib.GridmmLibraryError("gridmm ops need GPU tensors (got %s); no CPU fallback exists" % t.device)
        if t.device != hidden.device:
            raise ValueError("a tensor is on %s, hidden on %s" % (t.device, hidden.device))
    dt, ws = hidden.dtype, weight.shape
    if dt not in _DTYPES:
        raise ValueError("hidden is fp32, bf16 or fp16, not %s" % dt)
    if weight.dtype != dt:
        raise ValueError("weight is %s, hidden %s: one type for both" % (weight.dtype, dt))
    if hidden.dim() < 1 or len(ws) != 2 or ws[1] != hidden.shape[-1]:
        raise ValueError("hidden (..., K) and weight (V, K), not %s and %s" % (tuple(hidden.shape), tuple(ws)))
    if ws[0] < 1 or ws[1] < 1:
        raise ValueError("an empty weight %s" % (tuple(ws),))
    if ws[0] > MAX_VOCAB or ws[1] > MAX_HIDDEN or hidden.numel() > MAX_ROWS * ws[1]:
        raise ValueError("at most %d rows, %d of weight, %d hidden; not %s and %s" % (MAX_ROWS, MAX_VOCAB, MAX_HIDDEN,
                                                                                      tuple(hidden.shape), tuple(ws)))
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != ws[0]:
            raise ValueError("bias (V,), not %s" % (tuple(bias.shape),))
        if bias.dtype != torch.float32 and bias.dtype != dt:
            raise ValueError("bias is %s: fp32 or the weight's type" % bias.dtype)


def _apart(w, ld):
    """Rows that the tile products cannot read where they lie (16 bits: 16-byte boundaries, 32-bit offsets within a tile)."""
    return w.data_ptr() & 15 != 0 or ld % 8 != 0 or ld > 1 << 22


def _place(hidden, w, b, index):
    return (hidden.data_ptr(), w.data_ptr(), 0 if b is None else b.data_ptr(), index.data_ptr(), hidden.stride(0), w.stride(0), index.stride(0),
            hidden.numel(), w.numel(), index.numel())


def _moved(ctx, g, hidden, w, b, index, saved):
    """What saved-tensor hooks give back (checkpointing, offloading) are other tensors than the forward's, which may be gone: a descriptor
    with the addresses of these, and what it points to."""
    for t in (hidden, w, index, saved) + (() if b is None else (b,)):
        if t.device != g.device:
            raise RuntimeError("a tensor kept for the backward came back on %s, its gradient is on %s" % (t.device, g.device))
    d = _Desc.from_buffer_copy(ctx.desc)
    dt = hidden.dtype
    if ((tuple(hidden.shape), tuple(w.shape), index.numel()) != ((d.rows, d.hidden_size), (d.vocab, d.hidden_size), d.rows * max(d.slots, 1))
            or dt not in _DTYPES or _DTYPES[dt] != d.dtype or w.dtype != dt or index.dtype != (torch.int64 if d.index64 else torch.int32)
            or (b is not None and (b.numel() != d.vocab or _DTYPES.get(b.dtype) != d.bias_dtype))):
        raise RuntimeError("the tensors kept for the backward came back with other shapes or types")
    h, ldh = _rows(hidden)
    w, ldw = _rows(w)
    if not d.packed and _apart(w, ldw):          # (the forward read W where it lay)
        w, ldw = w.clone(memory_format=torch.contiguous_format), w.shape[1]
    if d.slots:
        index, ldi = _rows(index)
        d.ids, d.ld_ids = index.data_ptr(), max(ldi, d.slots)
    else:
        index = index.contiguous()
        d.labels = index.data_ptr()
    # (a single row: whatever its stride says)
    d.hidden, d.ld_hidden, d.weight, d.ld_weight = h.data_ptr(), max(ldh, d.hidden_size), w.data_ptr(), ldw
    if b is not None:
        b = b.contiguous()
        d.bias = b.data_ptr()
    return d, (h, w, b, index)


def _vocab_backward(ctx, g):
    if g is None:
        return (None,) * 8
    hidden, w, b, index, saved = ctx.saved_tensors
    d, keep = ctx.desc, None
    if _place(hidden, w, b, index) != ctx.place or not saved.is_cuda:
        d, keep = _moved(ctx, g, hidden, w, b, index, saved)
    if g.dtype != torch.float32:
        g = g.float()
    need_h, need_w, need_b = ctx.needs_input_grad[:3]
    n_ws, prm = ctx.n_ws, ctx.prm
    dh = hidden.new_empty(hidden.shape) if need_h else None
    dw = w.new_empty(w.shape) if need_w else None
    db = b.new_empty(b.shape) if need_b else None
    with _on(w.device):
        ws = saved.new_empty(n_ws)
        # (addresses as plain numbers: half the time of an object each)
        _lib.check(_lib.load().gridmm_vocab_loss_bwd(
            ctypes.byref(d), saved.data_ptr(), saved.numel(), g.data_ptr(), g.stride(0), dh.data_ptr() if need_h else None,
            dw.data_ptr() if need_w else None, db.data_ptr() if need_b else None, ws.data_ptr(), n_ws, _stream()), "gridmm_vocab_loss_bwd")
    return dh, DEFERRED.hand(prm[0], dw), DEFERRED.hand(prm[1], db), None, None, None, None, None


_vocab_backward_once = once_differentiable(_vocab_backward)


class _VocabLoss(torch.autograd.Function):
    """hidden (R, K), weight (V, K), bias (V,) or None, index (R,) labels or (R, S) ids, teacher None or (R, S) -> losses (R,)."""

    @staticmethod
    def forward(ctx, hidden, weight, bias, index, teacher, ignore_index, temperature, recording):
        lib = _lib.load()
        w, ldw = _rows(weight)
        b = None if bias is None else bias.contiguous()
        (R, K), V, dt = hidden.shape, w.shape[0], w.dtype
        S = 0 if teacher is None else index.shape[1]
        at, need = index.data_ptr(), recording and any(ctx.needs_input_grad[:3])
        # (a single row: whatever its stride says)
        d = _Desc(hidden.data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(), None if S else at, at if S else None,
                  teacher.data_ptr() if S else None, max(hidden.stride(0), K), ldw, max(index.stride(0), S) if S else 0,
                  max(teacher.stride(0), S) if S else 0, ignore_index, R, V, K, S, _DTYPES[dt], 0 if b is None else _DTYPES[b.dtype],
                  index.dtype == torch.int64, not need, _apart(w, ldw), temperature)
        ref = ctypes.byref(d)
        n_saved, n_ws = lib.gridmm_vocab_loss_saved_bytes(ref), lib.gridmm_vocab_loss_workspace(ref, 0)
        if n_saved == 0:
            raise ValueError("too many rows for this vocabulary or these slots (rows / 128 x vocabulary / 128 <= 2^23, rows x slots / 8 <= "
                             "2^25): rows %d, vocabulary %d, slots %d" % (R, V, S))
        loss = hidden.new_empty(R, dtype=torch.float32)
        saved = hidden.new_empty(n_saved, dtype=torch.uint8)
        ws = saved.new_empty(n_ws) if n_ws else None
        _lib.check(lib.gridmm_vocab_loss_fwd(ref, loss.data_ptr(), saved.data_ptr(), n_saved, ws.data_ptr() if n_ws else None, n_ws, _stream()),
                   "gridmm_vocab_loss_fwd")
        if need:
            ctx.set_materialize_grads(False)
            ctx.save_for_backward(hidden, w, b, index, saved)
            ctx.desc, ctx.place, ctx.n_ws = d, _place(hidden, w, b, index), lib.gridmm_vocab_loss_workspace(ref, 1)
            P = torch.nn.Parameter                   # (nothing else is kept alive here)
            ctx.prm = [weight if isinstance(weight, P) else None, bias if isinstance(bias, P) else None]
        return loss

    @staticmethod
    def backward(ctx, g):
        # (a backward that records itself: marked as once differentiable)
        return (_vocab_backward_once if torch.is_grad_enabled() else _vocab_backward)(ctx, g)


def vocab_cross_entropy(hidden, weight, labels, bias=None, ignore_index=-1):
    """Cross entropy of softmax(hidden weight^T + bias) against labels: fp32 losses of labels' shape, 0 where the label is
    ignore_index (those rows cost nothing and get no gradient).  hidden (..., K) and weight (V, K) in one of fp32 / bf16 / fp16,
    bias (V,) in that type or fp32, labels (...) int64 or int32.  Gradients of hidden, weight and bias in their types.

    A label outside [0, V) that is not ignore_index makes its row's loss NaN, and with it the gradients that it reaches.  A bias of -inf
    or of the type's lowest number takes its column out of the softmax; with no column left a row is NaN.  At most 2^20 rows, 2^27
    columns, and 2^37 scores.  fp32 rows (of hidden, or of weight) whose largest values are more than 2^14 apart, and fp32 and fp16 rows whose
    upstream gradients times largest values are more than 2^20 apart, keep their accuracy on slower matrix instructions: 5 to 7 times the time.

    Memory beside the results: what is kept for the backward is a copy of hidden, and one of weight where it is fp32 or cannot be read in
    place and takes at most 512 MB; the backward holds one piece of the scores' gradient at a time, of 512 MB, or of 32 KB a row where that is more
    (from 16384 rows on), fp32 sums of d_hidden (256 MB at most, or 4 bytes a value) and, fp32 and fp16, one more copy of hidden; the forward 8
    bytes for 128 columns of a row.  A few rows, and small heads, keep their scores (4 bytes each)."""
    _check_head(hidden, weight, bias, labels)
    if labels.shape != hidden.shape[:-1]:
        raise ValueError("labels %s for hidden %s" % (tuple(labels.shape), tuple(hidden.shape)))
    if labels.dtype != torch.int64 and labels.dtype != torch.int32:
        raise ValueError("labels are int64 or int32, not %s" % labels.dtype)
    with _on(hidden.device):
        if labels.dim() == 1:
            return _VocabLoss.apply(_rows(hidden)[0], weight, bias, labels.contiguous(), None, int(ignore_index), 1.0, torch.is_grad_enabled())
        y = labels.reshape(-1).contiguous()
        return _VocabLoss.apply(_rows(hidden)[0], weight, bias, y, None, int(ignore_index), 1.0, torch.is_grad_enabled()).view(labels.shape)


def vocab_distillation(hidden, weight, teacher_ids, teacher_logits, bias=None, temperature=1.0):
    """Distillation from a teacher's top logits over the same head: with p = softmax(teacher_logits / T) over the slots of a row and
    q = softmax((hidden weight^T + bias) / T) over the whole vocabulary, T^2 sum_s p_s (log p_s - log q[id_s]) as fp32 losses of
    hidden's leading shape.  teacher_ids (..., S) int64 or int32: an id < 0 is an empty slot, an id >= V makes its row NaN, ids may
    repeat; teacher_logits (..., S) (top_logits gives both).  A row without a filled slot above -inf: loss 0, no gradient.
    Gradients of hidden, weight and bias; the teacher gets none.  1e-6 <= T <= 1e6, at most 2^16 slots; sizes else as
    vocab_cross_entropy."""
    _check_head(hidden, weight, bias, teacher_ids, teacher_logits)
    _need(teacher_ids.dim() >= 1 and teacher_ids.shape == teacher_logits.shape
          and tuple(teacher_ids.shape[:-1]) == tuple(hidden.shape[:-1]) and teacher_ids.shape[-1] >= 1,
          "teacher_ids %s and teacher_logits %s for hidden %s" % (tuple(teacher_ids.shape), tuple(teacher_logits.shape),
                                                                  tuple(hidden.shape)))
    _need(teacher_ids.dtype in (torch.int64, torch.int32), "teacher_ids are int64 or int32, not %s" % teacher_ids.dtype)
    _need(teacher_logits.dtype in _DTYPES, "teacher_logits are fp32, bf16 or fp16, not %s" % teacher_logits.dtype)
    T = float(temperature)
    _need(1e-6 <= T <= 1e6, "a temperature of 1e-6 to 1e6, not %r" % (temperature,))
    _need(teacher_ids.shape[-1] <= MAX_SLOTS, "at most %d slots, not %d" % (MAX_SLOTS, teacher_ids.shape[-1]))
    with _on(hidden.device):
        h, _ = _rows(hidden)
        ids, _ = _rows(teacher_ids)
        t, _ = _rows(teacher_logits.detach().float())
        loss = _VocabLoss.apply(h, weight, bias, ids, t, -1, T, torch.is_grad_enabled())
        return loss if hidden.dim() == 2 else loss.view(hidden.shape[:-1])


def top_logits(logits, k):
    """The k largest of every row of logits (..., V): (values (..., k) in the logits' type, ids (..., k) int64, lse (...) fp32 = the
    row's log-sum-exp).  Sorted by value, among equal values by id (the lowest first; -0 equals +0), NaN before everything.
    1 <= k <= min(V, 1024).  No gradients: a teacher's scores."""
    if not logits.is_cuda:
        raise _lib.GridmmLibraryError("gridmm ops need GPU tensors (got %s); no CPU fallback exists" % logits.device)
    _need(logits.dtype in _DTYPES, "logits are fp32, bf16 or fp16, not %s" % logits.dtype)
    k = int(k)
    _need(logits.dim() >= 1 and 1 <= k <= min(logits.shape[-1], MAX_TOP), "1 <= k <= min(V, %d): k = %d of %s"
          % (MAX_TOP, k, tuple(logits.shape)))
    _need(logits.shape[-1] < 2 ** 31 and logits.numel() <= MAX_TOP_ROWS * logits.shape[-1], "at most %d rows of less than 2^31 logits, not %s"
          % (MAX_TOP_ROWS, tuple(logits.shape)))
    lib = _lib.load()
    with _on(logits.device):
        x, ld = _rows(logits.detach())
        lead, dev, R, V = logits.shape[:-1], logits.device, x.shape[0], x.shape[1]
        values = torch.empty(*lead, k, dtype=x.dtype, device=dev)
        ids = torch.empty(*lead, k, dtype=torch.int64, device=dev)
        lse = torch.empty(lead, dtype=torch.float32, device=dev)
        n = lib.gridmm_top_logits_workspace(R, V, k)
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        _lib.check(lib.gridmm_top_logits(_p(x), ld, _DTYPES[x.dtype], R, V, k, _p(values), _p(ids), _p(lse), _p(ws), n, _stream()),
                   "gridmm_top_logits")
    return values, ids, lse
