"""Operators between token ids and a model, on torch tensors: embedding lookup, next-token cross entropy and distillation over
the whole vocabulary, each with its gradient.

They take ids as `Tokenizer.encode_to_device` and `encode_batch_to_device` leave them on the GPU, run as kernels of
libgtok.so (`gtok_x_embed` and the entries after it in include/gtok.h, where the formulas are) on torch's current stream, and wait for
nothing.  Every call makes its own outputs and workspace by torch's allocator, so calls may be captured into CUDA graphs and may
run on several streams at once.

    ids, offsets = tokenizer.encode_batch_to_device(texts)
    hidden = model(embed(ids, table, scale=...))
    loss = cross_entropy(hidden, out_table, next_targets(ids, offsets))
    loss.backward()

`embed`, `cross_entropy` and `distill` take part in autograd.  `embed_grad`, `cross_entropy_forward`, `cross_entropy_grad`,
`distill_forward` and `distill_grad` are the same passes without autograd.  A step that is captured into a CUDA graph takes these: autograd's
nodes for the gradients of leaves belong to the stream that first used them, and a backward pass of torch's that is captured on
another one while they live fails.  There are no second and no forward-mode derivatives: the former raise in torch, and dual tensors are
refused.  torch.compile and torch.export do not look into the operators: compiled code calls them through torch.compiler.disable, between its
graphs.
"""
import ctypes
import struct

import torch
from torch.autograd import forward_ad

from . import GTokError, load_lib
from .ctypes_host import Matrix as _Matrix

__all__ = ["embed", "embed_grad", "next_targets", "cross_entropy", "cross_entropy_forward", "cross_entropy_grad", "distill", "distill_forward", "distill_grad"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_IDS = {torch.int32: 32, torch.int64: 64}
MAX_ENTRIES = 1024
_LEAST, _MOST = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max


class _Loss(ctypes.Structure):
    _fields_ = [("hidden", _Matrix), ("weight", _Matrix), ("targets", ctypes.c_void_p), ("target_stride", ctypes.c_int64),
                ("target_bits", ctypes.c_int32), ("entries", ctypes.c_int32), ("teacher_logits", _Matrix), ("ignore", ctypes.c_int64),
                ("temperature", ctypes.c_float), ("mean", ctypes.c_int32), ("losses", ctypes.c_void_p), ("lse", ctypes.c_void_p),
                ("total", ctypes.c_void_p), ("grad", ctypes.c_void_p), ("grad_stride", ctypes.c_int64), ("d_hidden", _Matrix),
                ("d_weight", _Matrix), ("kept", ctypes.c_void_p), ("kept_bytes", ctypes.c_uint64), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_uint64), ("cuda_stream", ctypes.c_void_p)]


_HEAD = struct.Struct("@" + 2 * "Pqqqi" + "PqiiPqqqiqf")        # _Loss up to the temperature; what follows is 0 until it is set


_bound = None


def _lib():
    global _bound
    if _bound is None:
        lib = load_lib()
        vp, i32, i64, u64, mat = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.POINTER(_Matrix)
        lib.gtok_x_embed.restype = i32
        lib.gtok_x_embed.argtypes = [vp, i32, i64, mat, ctypes.c_float, mat, vp]
        lib.gtok_x_embed_grad_workspace.restype = i64
        lib.gtok_x_embed_grad_workspace.argtypes = [i64, i64, i64]
        lib.gtok_x_embed_grad.restype = i32
        lib.gtok_x_embed_grad.argtypes = [vp, i32, i64, mat, ctypes.c_float, mat, i32, vp, u64, vp]
        lib.gtok_x_next_targets.restype = i32
        lib.gtok_x_next_targets.argtypes = [vp, i64, vp, i64, vp, i32, vp, vp]
        lib.gtok_x_vocab_loss_workspace.restype = i64
        lib.gtok_x_vocab_loss_workspace.argtypes = [ctypes.POINTER(_Loss), i32]
        lib.gtok_x_vocab_loss_kept.restype = i64
        lib.gtok_x_vocab_loss_kept.argtypes = [ctypes.POINTER(_Loss)]
        for f in (lib.gtok_x_vocab_loss_forward, lib.gtok_x_vocab_loss_backward):
            f.restype = i32
            f.argtypes = [ctypes.POINTER(_Loss)]
        _bound = lib
    return _bound


def _done(code, what):
    if code < 0:
        raise GTokError("%s returned %d: %s" % (what, code, _bound.gtok_x_last_error().decode("utf-8", "replace")))
    return code


def _on_gpu(first, **others):
    """Index of the GPU that all of them are on."""
    try:
        index = first.get_device()
        for t in others.values():
            if not (t.is_cuda and t.get_device() == index and t.layout is torch.strided):
                break
        else:
            return index
    except (AttributeError, RuntimeError):
        pass
    for name, t in others.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s must be a torch tensor" % name)
        if t.layout is not torch.strided:
            raise TypeError("%s must be a dense tensor" % name)
    device = getattr(first, "device", None)
    for name, t in others.items():
        if t.device != device:
            raise ValueError("%s is on %s, other arguments on %s" % (name, t.device, device))
    raise ValueError("tensors must be on the GPU, not on %s" % device)


def _no_tangents(*tensors):
    """A result without the tangent that it should have would be taken for a constant."""
    if getattr(forward_ad, "_current_level", 0) < 0:         # outside of all levels no tensor has one
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("the vocabulary operators have no forward-mode derivatives")


def _there(index, f, *args):
    """f(*args) with GPU `index` current."""
    if torch.cuda.current_device() == index:
        return f(*args)
    with torch.cuda.device(index):
        return f(*args)


def _ids_of(name, t):
    if t.dtype not in _IDS:
        raise TypeError("%s must be int32 or int64, not %s" % (name, t.dtype))
    return t if t.is_contiguous() else t.contiguous()


def _rows(t):
    """`t` with its rows' elements next to one another and in memory as they are (a copy only where they are not)."""
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _parts(t):
    rows, cols = t.shape
    return t.data_ptr(), rows, cols, t.stride(0) if rows > 1 else cols, _TYPES[t.dtype]


def _matrix(t):
    return _Matrix(*_parts(t))


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)       # (a tenth of the time of the public way)


def _stream(index):
    return _raw_stream(index) if _raw_stream else torch.cuda.current_stream(index).cuda_stream


def _scale(scale):
    scale = float(scale)
    if not -_MOST <= scale <= _MOST:
        raise ValueError("scale must be finite, in float32")
    return scale


# ---- embedding -------------------------------------------------------------------
def _table(name, t):
    if t.dim() != 2:
        raise ValueError("%s must have two dimensions" % name)
    if t.dtype not in _TYPES:
        raise TypeError("%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))
    if t.shape[1] < 1:
        raise ValueError("%s must have columns" % name)


def _embed(ids, table, scale, index):
    flat, rows = _ids_of("ids", ids), _rows(table)
    vocab, width = table.shape
    out = table.new_empty((*ids.shape, width))
    code = _lib().host.embed(flat.data_ptr(), _IDS[flat.dtype], flat.numel(), rows.data_ptr(), vocab, width, rows.stride(0) if vocab > 1 else width,
                             _TYPES[table.dtype], scale, out.data_ptr(), _stream(index))
    if code:
        _done(code, "gtok_x_embed")
    return out


class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, table, scale):
        ctx.save_for_backward(ids)
        ctx.vocab, ctx.scale = table.shape[0], scale
        return _there(table.get_device(), _embed, ids, table, scale, table.get_device())

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        ids, = ctx.saved_tensors
        return None, embed_grad(ids, grad, ctx.vocab, scale=ctx.scale), None


def embed(ids, table, scale=1.0):
    """Rows of `table` [vocab, width] (float32, bfloat16 or float16) by id, times `scale`: a tensor of ids.shape + (width,).

    ids: int32 or int64, any shape.  A negative id gives a row of zeros, one beyond the table a row of NaN; neither has a gradient."""
    _no_tangents(table)
    index = _on_gpu(table, table=table, ids=ids)
    _table("table", table)
    scale = _scale(scale)
    if table.requires_grad and torch.is_grad_enabled():
        return _Embed.apply(ids, table, scale)
    return _there(index, _embed, ids, table, scale, index)


def _overlap(a, b):
    """Whether two matrices of one type may share an element: their memory does, and not as columns beside one another."""
    size = a.element_size()
    at = [t.data_ptr() for t in (a, b)]
    end = [x + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * size for x, t in zip(at, (a, b))]
    if not (a.numel() and b.numel() and at[0] < end[1] and at[1] < end[0]):
        return False
    line = (a if a.shape[0] > 1 else b).stride(0) * size
    apart = (at[1] - at[0]) % line if line else 0
    alike = a.shape[0] == 1 or b.shape[0] == 1 or a.stride(0) == b.stride(0)
    return not (alike and a.shape[1] * size <= apart <= line - b.shape[1] * size)


def embed_grad(ids, grad, vocab, scale=1.0, out=None, accumulate=False):
    """Gradient of `embed`: [vocab, width] with, for each id, `scale` times the sum of the rows of `grad` (ids.shape + (width,)) that were
    looked up from it, 0 for ids that were not.  The sum is in float32 and in the order of the ids, whatever they are.

    out: where to write it, of grad's type and apart from grad's memory.  With `accumulate` it is added to what `out` holds, as for a table that is an
    output table too, and rows that are not asked for are not touched."""
    _no_tangents(grad, out)
    index = _on_gpu(grad, grad=grad, ids=ids)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape:
        raise ValueError("grad must have the shape of ids and one dimension more")
    width, vocab = grad.shape[-1], int(vocab)
    flat = _ids_of("ids", ids)
    rows = _rows(grad if grad.dim() == 2 else grad.reshape(flat.numel(), width))
    _table("grad", rows)
    if vocab < 0:
        raise ValueError("vocab must not be negative")
    if accumulate and out is None:
        raise ValueError("accumulate needs `out`")
    scale = _scale(scale)
    if out is not None:
        _on_gpu(grad, out=out)
        if out.shape != (vocab, width) or out.dtype != grad.dtype or (width > 1 and out.stride(1) != 1) or out.is_neg():
            raise ValueError("out must be [vocab, width] of grad's type with the elements of a row next to one another, no view of negated ones")
        if _overlap(rows, out):
            raise ValueError("out and grad overlap")
    result = _there(index, _embed_grad, flat, rows, vocab, scale, out, accumulate, index)
    if out is not None:
        torch.autograd.graph.increment_version(out)         # who has saved it for a backward pass is to notice
    return result


def _embed_grad(flat, rows, vocab, scale, out, accumulate, index):
    lib, n, width = _lib(), flat.numel(), rows.shape[1]
    if out is None:
        out = rows.new_empty((vocab, width))
    need = _done(lib.gtok_x_embed_grad_workspace(n, vocab, width), "gtok_x_embed_grad_workspace")
    work = torch.empty(need, dtype=torch.uint8, device=rows.device)
    _done(lib.gtok_x_embed_grad(flat.data_ptr(), _IDS[flat.dtype], n, _matrix(rows), scale, _matrix(out), bool(accumulate), work.data_ptr(), need,
                                _stream(index)), "gtok_x_embed_grad")
    return out


# ---- targets ---------------------------------------------------------------------
def next_targets(ids, offsets, loss_mask=None, ignore_index=-100):
    """For packed documents as `Tokenizer.encode_batch_to_device` gives them (int32 ids, int32 n + 1 offsets): the id that follows each
    position in its document, `ignore_index` at a document's last position, outside of all documents, and where the boolean
    `loss_mask` (same length as ids) is false.  int32."""
    index = _on_gpu(ids, ids=ids, offsets=offsets)
    if ids.dtype != torch.int32 or ids.dim() != 1 or offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError("ids and offsets must be one-dimensional and int32, offsets not empty")
    if not -(1 << 31) <= ignore_index < 0:
        raise ValueError("ignore_index must be negative, in 32 bits")
    if loss_mask is not None:
        _on_gpu(ids, loss_mask=loss_mask)
        if loss_mask.dtype != torch.bool or loss_mask.shape != ids.shape:
            raise ValueError("loss_mask must be boolean and as long as ids")
        loss_mask = loss_mask.contiguous()
    return _there(index, _next_targets, ids.contiguous(), offsets.contiguous(), loss_mask, int(ignore_index), index)


def _next_targets(ids, offsets, mask, ignore_index, index):
    out = torch.empty_like(ids)
    _done(_lib().gtok_x_next_targets(ids.data_ptr(), ids.numel(), offsets.data_ptr(), offsets.numel() - 1, mask.data_ptr() if mask is not None else None,
                                     ignore_index, out.data_ptr(), _stream(index)), "gtok_x_next_targets")
    return out


# ---- losses over the vocabulary -----------------------------------------------------
def _flat(hidden):
    return _rows(hidden if hidden.dim() == 2 else hidden.reshape(hidden.shape[:-1].numel(), hidden.shape[-1]))


def _lines(weight):
    """`weight` with rows that do not lie over one another."""
    weight = _rows(weight)
    return weight.contiguous() if weight.stride(0) < weight.shape[1] and weight.shape[0] > 1 else weight


class _Call:
    """Arguments of one loss, checked, and what keeps their memory alive.  `teacher_logits` is None for cross entropy."""

    def __init__(self, hidden, weight, ids, teacher_logits, ignore_index, temperature):
        _no_tangents(hidden, weight)
        if teacher_logits is None:
            what, lead = "targets", getattr(ids, "shape", None)
            self.index = _on_gpu(hidden, hidden=hidden, weight=weight, targets=ids)
        else:
            what, lead = "teacher_ids", getattr(ids, "shape", (None,))[:-1]
            self.index = _on_gpu(hidden, hidden=hidden, weight=weight, teacher_ids=ids, teacher_logits=teacher_logits)
            if ids.dim() < 1 or teacher_logits.shape != ids.shape or not 1 <= ids.shape[-1] <= MAX_ENTRIES:
                raise ValueError("teacher_ids and teacher_logits must be [..., k] with k from 1 to %d" % MAX_ENTRIES)
            if teacher_logits.dtype not in _TYPES:
                raise TypeError("teacher_logits must be float32, bfloat16 or float16, not %s" % teacher_logits.dtype)
        if hidden.dtype not in (torch.bfloat16, torch.float16) or weight.dtype != hidden.dtype:
            raise TypeError("hidden and weight must both be bfloat16 or both float16, not %s and %s" % (hidden.dtype, weight.dtype))
        if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or 0 in weight.shape:
            raise ValueError("hidden must be [..., width] and weight [vocab, width]")
        if hidden.shape[:-1] != lead:
            raise ValueError("hidden and %s differ in their leading dimensions" % what)
        temperature = float(temperature)
        if not _LEAST <= temperature <= _MOST:
            raise ValueError("temperature must be positive and finite, as a normal number of float32")
        # (kept until the kernels are queued: memory that is let go before may be handed out again to the same call)
        self.hidden, self.weight, self.ids = h, w, i = _flat(hidden), _lines(weight), _ids_of(what, ids)
        self.n, kind, bits = h.shape[0], _TYPES[h.dtype], _IDS[i.dtype]
        k, logits = 0, (0, 0, 0, 0, 0)
        if teacher_logits is not None:
            k, self.logits = ids.shape[-1], _flat(teacher_logits)
            logits = _parts(self.logits)
        memory = bytearray(ctypes.sizeof(_Loss))
        _HEAD.pack_into(memory, 0, *_parts(h), *_parts(w), i.data_ptr(), k, bits, k, *logits, ignore_index, temperature)
        self.args = _Loss.from_buffer(memory)

    def let_go(self):
        """Forgets the tensors, for a call that waits for its backward pass; `again` is that pass's."""
        self.hidden = self.ids = self.logits = self.weight = self.kept = self.work = None

    def again(self, weight, kept):
        call = object.__new__(_Call)
        call.index, call.n, call.args, call.weight, call.kept = self.index, self.n, _Loss.from_buffer_copy(self.args), _lines(weight), kept
        a = call.args
        a.weight, a.kept = _matrix(call.weight), kept.data_ptr()
        a.lse = kept.data_ptr() + a.kept_bytes
        return call

    def _run(self, entry, backward, more=0):
        """`more`: bytes behind the workspace, whose address is returned."""
        a = self.args
        need = (_done(_lib().gtok_x_vocab_loss_workspace(a, backward), "gtok_x_vocab_loss_workspace") + 255) & ~255
        self.work = torch.empty(need + more, dtype=torch.uint8, device=self.weight.device)
        at = self.work.data_ptr()
        a.workspace, a.workspace_bytes, a.cuda_stream = at, need, _stream(self.index)
        if more:
            if not a.losses:
                a.losses = at + need
            if not a.lse:
                a.lse = at + need + more // 2
        _done(entry(a), entry.__name__)

    def forward(self, reduction, keep=False, want_lse=False):
        return _there(self.index, self._forward, reduction, keep, want_lse)

    def _forward(self, reduction, keep, want_lse):
        """(loss, lse or None).  With `keep`, what the backward pass takes is in `self.kept`, lse behind it; losses and lse that nobody asks for
        lie behind the workspace."""
        a, n, device, lse = self.args, self.n, self.weight.device, None
        if reduction == "none":
            result = torch.empty(n, dtype=torch.float32, device=device)
            a.losses = result.data_ptr()
        else:
            result = torch.empty((), dtype=torch.float32, device=device)
            a.total, a.mean = result.data_ptr(), reduction == "mean"
        if keep:
            size = (_done(_lib().gtok_x_vocab_loss_kept(a), "gtok_x_vocab_loss_kept") + 255) & ~255
            self.kept = torch.empty(size + 4 * n, dtype=torch.uint8, device=device)
            a.kept, a.kept_bytes, a.lse = self.kept.data_ptr(), size, self.kept.data_ptr() + size
        elif want_lse:
            lse = torch.empty(n, dtype=torch.float32, device=device)
            a.lse = lse.data_ptr()
        self._run(_lib().gtok_x_vocab_loss_forward, 0, 8 * n)
        return result, lse

    def backward(self, lse, grad, reduction, want_hidden, want_weight):
        """`lse`: None where it lies behind what was kept."""
        return _there(self.index, self._backward, lse, grad, reduction, want_hidden, want_weight)

    def _backward(self, lse, grad, reduction, want_hidden, want_weight):
        a = self.args
        if lse is not None:
            lse = lse.resolve_neg().contiguous()
            a.lse = lse.data_ptr()
        grad = grad.resolve_neg()
        if reduction == "none":
            grad = grad if grad.dim() == 1 else grad.reshape(-1)
            a.grad_stride = grad.stride(0) if grad.numel() > 1 else 0
        a.grad, a.mean = grad.data_ptr(), reduction == "mean"
        d_hidden = d_weight = None
        if want_hidden:
            d_hidden = self.weight.new_empty((self.n, self.weight.shape[1]))
            a.d_hidden = _matrix(d_hidden)
        if want_weight:
            d_weight = self.weight.new_empty(self.weight.shape)
            a.d_weight = _matrix(d_weight)
        self._run(_lib().gtok_x_vocab_loss_backward, 1)
        return d_hidden, d_weight


def _check_reduction(reduction):
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none'")


def _check_grad(lse, grad, lead, reduction, hidden):
    _check_reduction(reduction)
    _on_gpu(hidden, lse=lse, grad=grad)
    if lse.dtype != torch.float32 or grad.dtype != torch.float32:
        raise TypeError("lse and grad must be float32")
    if lse.shape != lead or grad.shape != (lead if reduction == "none" else ()):
        raise ValueError("lse must have the targets' shape, grad that of the loss")


class _LossFunction(torch.autograd.Function):
    """Keeps the forward pass's copy of the rows that have a loss in place of the hidden states."""

    @staticmethod
    def forward(ctx, call, hidden, weight, reduction):
        loss, _ = call.forward(reduction, keep=True)
        ctx.save_for_backward(weight, call.kept)
        ctx.call, ctx.reduction, ctx.shape = call, reduction, hidden.shape
        call.let_go()
        return loss.view(hidden.shape[:-1]) if reduction == "none" else loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        _no_tangents(grad)
        weight, kept = ctx.saved_tensors
        _, want_hidden, want_weight, _ = ctx.needs_input_grad
        d_hidden, d_weight = ctx.call.again(weight, kept).backward(None, grad, ctx.reduction, want_hidden, want_weight)
        return None, d_hidden.view(ctx.shape) if want_hidden else None, d_weight, None


def _loss(hidden, weight, ids, teacher_logits, reduction, ignore_index, temperature):
    _check_reduction(reduction)
    call = _Call(hidden, weight, ids, teacher_logits, ignore_index, temperature)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LossFunction.apply(call, hidden, weight, reduction)
    loss, _ = call.forward(reduction)
    return loss.view(hidden.shape[:-1]) if reduction == "none" else loss


def cross_entropy(hidden, weight, targets, reduction="mean", ignore_index=-100, temperature=1.0):
    """Softmax cross entropy of the logits hidden @ weight.T / temperature against `targets`, without holding the logits.

    hidden: [..., width], weight: [vocab, width], both bfloat16 or both float16; targets: int32 or int64 of hidden's leading shape.
    Targets of `ignore_index`, or negative, carry no loss and no gradient; a target beyond the vocabulary gives NaN.
    reduction: 'none' (float32 of the targets' shape), 'sum', or 'mean' over the rows that carry a loss (0 where none does)."""
    return _loss(hidden, weight, targets, None, reduction, ignore_index, temperature)


def cross_entropy_forward(hidden, weight, targets, reduction="none", ignore_index=-100, temperature=1.0):
    """(loss, lse): what `cross_entropy` returns and the float32 logarithms of the rows' sums, which `cross_entropy_grad` takes."""
    _check_reduction(reduction)
    loss, lse = _Call(hidden, weight, targets, None, ignore_index, temperature).forward(reduction, want_lse=True)
    return (loss.view(targets.shape) if reduction == "none" else loss), lse.view(targets.shape)


def cross_entropy_grad(hidden, weight, targets, lse, grad, reduction="none", ignore_index=-100, temperature=1.0, want_hidden=True, want_weight=True):
    """(d_hidden, d_weight) for the gradient `grad` of the loss (float32, of its shape); None for what is not wanted."""
    _no_tangents(lse, grad)
    call = _Call(hidden, weight, targets, None, ignore_index, temperature)
    _check_grad(lse, grad, targets.shape, reduction, hidden)
    d_hidden, d_weight = call.backward(lse, grad, reduction, want_hidden, want_weight)
    return d_hidden.view(hidden.shape) if d_hidden is not None else None, d_weight


def distill(hidden, weight, teacher_ids, teacher_logits, temperature=1.0, reduction="mean"):
    """Divergence of a student's softmax from a teacher's top logits, both over `temperature`, without holding the student's logits.

    hidden, weight: as in `cross_entropy`.  teacher_ids (int32 or int64) and teacher_logits: [..., k], k up to 1024, in any order;
    a negative id is no entry.  The teacher's probabilities are the softmax over a row's entries; a row without any carries no loss.
    The customary factor temperature ** 2 is not applied.  There is no gradient for the teacher."""
    _no_tangents(hidden, weight)
    _on_gpu(hidden, teacher_logits=teacher_logits)
    return _loss(hidden, weight, teacher_ids, teacher_logits, reduction, -100, temperature)


def distill_forward(hidden, weight, teacher_ids, teacher_logits, temperature=1.0, reduction="none"):
    """(loss, lse), as `cross_entropy_forward`."""
    _check_reduction(reduction)
    _no_tangents(hidden, weight)
    _on_gpu(hidden, teacher_logits=teacher_logits)
    loss, lse = _Call(hidden, weight, teacher_ids, teacher_logits, -100, temperature).forward(reduction, want_lse=True)
    lead = hidden.shape[:-1]
    return (loss.view(lead) if reduction == "none" else loss), lse.view(lead)


def distill_grad(hidden, weight, teacher_ids, teacher_logits, lse, grad, temperature=1.0, reduction="none", want_hidden=True, want_weight=True):
    """(d_hidden, d_weight), as `cross_entropy_grad`."""
    _no_tangents(hidden, weight, lse, grad)
    _on_gpu(hidden, teacher_logits=teacher_logits)
    call = _Call(hidden, weight, teacher_ids, teacher_logits, -100, temperature)
    _check_grad(lse, grad, hidden.shape[:-1], reduction, hidden)
    d_hidden, d_weight = call.backward(lse, grad, reduction, want_hidden, want_weight)
    return d_hidden.view(hidden.shape) if d_hidden is not None else None, d_weight
