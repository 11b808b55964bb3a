"""Operators from a model's last hidden states to the ids that it answers with, on torch tensors: products with an output table in 4 bits,
penalties, biases and grammar masks on logits, and the draw of an id for each row.

They are the other end of `vocab_ops`: kernels of libgtok.so (`gtok_x_table4_bytes` and the entries after it in include/gtok.h, where the formulas are)
on torch's current stream, that wait for nothing.  Every call makes its own outputs by torch's allocator, so calls may be captured into CUDA graphs and may run on
several streams at once.

    table = quantize_table(out_table)                          # once
    logits = table_logits(hidden, table)                       # a step: a hidden state for each request
    adjust_logits(logits, ids, offsets, repetition=1.1, out=logits)
    new, logprobs = sample(logits, torch.rand(len(logits), device="cuda"), temperature=0.8, top_p=0.95)
    for answer, i in zip(answers, new.tolist()):
        answer += [i] if i >= 0 else []                        # (-1: nothing was allowed)
    text = tokenizer.decode(answers[0])                        # of a whole one; a part may end within a character: decode_bytes

None of them has a gradient: where one would be asked for, by logits, hidden states, biases, penalties or wishes, they refuse, as they do for dual tensors.  A table in 4 bits is a constant:
weights and scales that it is made of may require a gradient, and get none from it.  torch.compile and torch.export do not look into the operators:
compiled code calls them through torch.compiler.disable, between its graphs.
"""
import ctypes
import struct

import torch

from .vocab_ops import _IDS, _LEAST, _MOST, _TYPES, _Matrix, _ids_of, _matrix, _no_tangents, _on_gpu, _overlap, _parts, _rows, _stream, _there, GTokError, load_lib

__all__ = ["QuantizedTable", "pack_table", "quantize_table", "table_logits", "adjust_logits", "sample"]

MAX_BIASES = 1024


class _Table4(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("bytes", ctypes.c_uint64), ("vocab", ctypes.c_int64), ("width", ctypes.c_int64), ("group", ctypes.c_int64),
                ("type", ctypes.c_int32), ("zeros", ctypes.c_int32)]


class _Adjustment(ctypes.Structure):
    _fields_ = [("logits", _Matrix), ("out", _Matrix), ("ids", ctypes.c_void_p), ("n_ids", ctypes.c_int64), ("id_bits", ctypes.c_int32), ("entries", ctypes.c_int32),
                ("offsets", ctypes.c_void_p), ("prompt_lengths", ctypes.c_void_p), ("repetition", ctypes.c_void_p), ("presence", ctypes.c_void_p),
                ("frequency", ctypes.c_void_p), ("one_repetition", ctypes.c_float), ("one_presence", ctypes.c_float), ("one_frequency", ctypes.c_float),
                ("reserved", ctypes.c_int32), ("bias_ids", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("bias_stride", ctypes.c_int64), ("allowed", ctypes.c_void_p),
                ("allowed_rows", ctypes.c_void_p), ("allowed_count", ctypes.c_int64), ("allowed_stride", ctypes.c_int64), ("cuda_stream", ctypes.c_void_p)]


class _Draw(ctypes.Structure):
    _fields_ = [("logits", _Matrix), ("u", ctypes.c_void_p), ("u_bits", ctypes.c_int32), ("one_top_k", ctypes.c_int32), ("temperature", ctypes.c_void_p),
                ("top_k", ctypes.c_void_p), ("top_p", ctypes.c_void_p), ("min_p", ctypes.c_void_p), ("one_temperature", ctypes.c_float), ("one_top_p", ctypes.c_float),
                ("one_min_p", ctypes.c_float), ("reserved", ctypes.c_int32), ("ids", ctypes.c_void_p), ("logprobs", ctypes.c_void_p), ("cuda_stream", ctypes.c_void_p)]


_ADJUSTMENT = struct.Struct("@" + 2 * "Pqqqi" + "PqiiPPPPPfffiPPqPPqqP")      # the structs at once: a fifth of the time of field by field
_DRAW = struct.Struct("@PqqqiPiiPPPPfffiPPP")


_bound = None


def _lib():
    global _bound
    if _bound is None:
        lib = load_lib()
        vp, i32, i64, mat, tab = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.POINTER(_Matrix), ctypes.POINTER(_Table4)
        lib.gtok_x_table4_bytes.restype = i64
        lib.gtok_x_table4_bytes.argtypes = [i64, i64, i64, i32]
        lib.gtok_x_table4_pack.restype = i32
        lib.gtok_x_table4_pack.argtypes = [tab, vp, i64, mat, vp, i64, vp]
        lib.gtok_x_table4_quantize.restype = i32
        lib.gtok_x_table4_quantize.argtypes = [tab, mat, vp]
        lib.gtok_x_table4_logits.restype = i32
        lib.gtok_x_table4_logits.argtypes = [mat, tab, mat, vp]
        lib.gtok_x_adjust_logits.restype = i32
        lib.gtok_x_adjust_logits.argtypes = [ctypes.POINTER(_Adjustment)]
        lib.gtok_x_sample.restype = i32
        lib.gtok_x_sample.argtypes = [ctypes.POINTER(_Draw)]
        _bound = lib
    return _bound


def _done(code, what):
    if code < 0:
        raise GTokError("%s returned %d: %s" % (what, code, _lib().gtok_x_last_error().decode("utf-8", "replace")))
    return code


def _no_gradient(what, *tensors):
    _no_tangents(*tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                raise NotImplementedError("%s has no gradient: call it under torch.no_grad() or on detached tensors" % what)


# ---- tables in 4 bits -------------------------------------------------------------
class QuantizedTable:
    """A table [vocab, width] in 4 bits, as `quantize_table` and `pack_table` make it: a scale in `dtype` (bfloat16 or float16), and with `zeros` a
    zero, for every `group` columns of a row.  It lies in `data`, one uint8 tensor, in an order of its own; `to`, copy.deepcopy, torch.save and (where this module has been
    imported) torch.load work as on tensors."""

    def __init__(self, vocab, width, group, dtype, zeros, device, data=None):
        self.vocab, self.width, self.group, self.dtype, self.zeros = vocab, width, group, dtype, zeros
        need = _done(_lib().gtok_x_table4_bytes(vocab, width, group, zeros), "gtok_x_table4_bytes")
        if data is None:
            data = torch.empty(need, dtype=torch.uint8, device=device)
        elif data.shape != (need,) or data.dtype != torch.uint8 or not data.is_contiguous():
            raise ValueError("data must be uint8 [%d]" % need)
        self._data = data
        self._args = _Table4(data.data_ptr(), need, vocab, width, group, _TYPES[dtype], zeros)

    @property
    def data(self):
        return self._data

    @property
    def device(self):
        return self._data.device

    def to(self, device):
        """The same table on another device."""
        data = self._data.to(device)
        return self if data is self._data else QuantizedTable(self.vocab, self.width, self.group, self.dtype, self.zeros, data.device, data)

    def __reduce__(self):                  # (copies and files: the address is not part of it)
        return QuantizedTable, (self.vocab, self.width, self.group, self.dtype, self.zeros, None, self._data)

    def __deepcopy__(self, memo):
        return QuantizedTable(self.vocab, self.width, self.group, self.dtype, self.zeros, None, self._data.clone())

    @property
    def shape(self):
        return torch.Size((self.vocab, self.width))

    def __repr__(self):
        return "QuantizedTable(%d x %d, group=%d, dtype=%s, zeros=%s, device=%s)" % (self.vocab, self.width, self.group, self.dtype, self.zeros, self.device)


torch.serialization.add_safe_globals([QuantizedTable])         # torch.load makes one from its sizes and its memory, which are looked at, and nothing else


def _group(group):
    group = int(group)
    if group != 32 and (group < 64 or group > 1 << 16 or group % 64):
        raise ValueError("group must be 32 or a multiple of 64, up to 65536")
    return group


def _table_shape(name, t):
    if t.dim() != 2 or 0 in t.shape or t.shape[0] > 1 << 24 or t.shape[1] > 1 << 16:
        raise ValueError("%s must be [vocab, width], up to 2^24 by 2^16 and not empty" % name)


def pack_table(codes, scales, zeros=None, group=128):
    """A `QuantizedTable` of codes that are there already: uint8 [vocab, width], 0 to 15 (of larger ones the low four bits count); scales: bfloat16 or float16
    [vocab, ceil(width / group)]; zeros: uint8 of the scales' shape, 8 everywhere where there are none.  An element stands for scale * (code - zero)."""
    group = _group(group)
    index = _on_gpu(codes, codes=codes, scales=scales, **({} if zeros is None else {"zeros": zeros}))
    _table_shape("codes", codes)
    if codes.dtype != torch.uint8 or (zeros is not None and zeros.dtype != torch.uint8):
        raise TypeError("codes and zeros must be uint8")
    if scales.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("scales must be bfloat16 or float16, not %s" % scales.dtype)
    vocab, width = codes.shape
    _no_tangents(scales)
    if scales.shape != (vocab, -(-width // group)) or (zeros is not None and zeros.shape != scales.shape):
        raise ValueError("scales and zeros must be [vocab, ceil(width / group)]")
    return _there(index, _pack, _rows(codes), _rows(scales.detach()), None if zeros is None else _rows(zeros), group, index)


def _pack(codes, scales, zeros, group, index):
    table = QuantizedTable(*codes.shape, group, scales.dtype, zeros is not None, codes.device)
    _done(_lib().gtok_x_table4_pack(table._args, codes.data_ptr(), codes.stride(0), _matrix(scales), None if zeros is None else zeros.data_ptr(),
                                    0 if zeros is None else zeros.stride(0), _stream(index)), "gtok_x_table4_pack")
    return table


def quantize_table(weight, group=128, zeros=False, dtype=None):
    """A `QuantizedTable` of `weight` [vocab, width] (float32, bfloat16 or float16), rounded to the nearest of 16 values a group: of 15 on both sides of 0, or with `zeros` of
    16 between the group's least and largest, 0 among them.  dtype: of the scales and of the hidden states to come, weight's by default (bfloat16 for float32).
    A group with a NaN, an infinity or more than its scale's type can say gives NaN."""
    group = _group(group)
    index = _on_gpu(weight, weight=weight)
    _table_shape("weight", weight)
    if weight.dtype not in _TYPES:
        raise TypeError("weight must be float32, bfloat16 or float16, not %s" % weight.dtype)
    if dtype is None:
        dtype = torch.bfloat16 if weight.dtype == torch.float32 else weight.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("dtype must be bfloat16 or float16")
    _no_tangents(weight)
    return _there(index, _quantize, _rows(weight.detach()), group, bool(zeros), dtype, index)


def _quantize(weight, group, zeros, dtype, index):
    table = QuantizedTable(*weight.shape, group, dtype, zeros, weight.device)
    _done(_lib().gtok_x_table4_quantize(table._args, _matrix(weight), _stream(index)), "gtok_x_table4_quantize")
    return table


def table_logits(hidden, table, dtype=torch.float32):
    """hidden @ table.T for a `QuantizedTable`: hidden [..., width] of the table's dtype, logits [..., vocab] in float32 or in that dtype.

    Made for the few rows of a decoding step.  No weight is rounded to 16 bits on the way; sums are in float32.  There is no gradient."""
    if table.__class__ is not QuantizedTable and not isinstance(table, QuantizedTable):
        raise TypeError("table must be a QuantizedTable, as quantize_table and pack_table make it")
    _no_gradient("table_logits", hidden)
    index = _on_gpu(hidden, hidden=hidden, table=table._data)
    if hidden.dtype != table.dtype:
        raise TypeError("hidden must be %s, as the table's scales are, not %s" % (table.dtype, hidden.dtype))
    if hidden.dim() < 1 or hidden.shape[-1] != table.width:
        raise ValueError("hidden must be [..., %d]" % table.width)
    if dtype != torch.float32 and dtype != table.dtype:
        raise TypeError("logits are float32 or %s" % table.dtype)
    return _there(index, _logits, hidden, table, dtype, index)


def _logits(hidden, table, dtype, index):
    flat = _rows(hidden if hidden.dim() == 2 else hidden.reshape(hidden.shape[:-1].numel(), hidden.shape[-1]))
    out = torch.empty((*hidden.shape[:-1], table.vocab), dtype=dtype, device=hidden.device)
    n = flat.shape[0]
    if n > 8 and (flat.data_ptr() % 16 or flat.stride(0) % 8):       # more rows are copied by whole 16 bytes
        width = flat.shape[1]
        flat = torch.empty((n, -(-width // 8) * 8), dtype=flat.dtype, device=flat.device)[:, :width].copy_(flat)
    if n:
        code = _lib().gtok_x_table4_logits(_matrix(flat), table._args, _Matrix(out.data_ptr(), n, table.vocab, table.vocab, _TYPES[dtype]), _stream(index))
        if code:
            _done(code, "gtok_x_table4_logits")
    return out


# ---- logits -----------------------------------------------------------------------
def _logits_of(logits):
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= 1 << 24:
        raise ValueError("logits must be [n, vocab] with 1 to 2^24 ids")
    if logits.shape[0] > 1 << 20:
        raise ValueError("logits must have at most 2^20 rows")
    if logits.dtype not in _TYPES:
        raise TypeError("logits must be float32, bfloat16 or float16, not %s" % logits.dtype)


def _pointer(name, t, dtype, shape, index, keep):
    """Address of `t`, one element next to the other, with what keeps its memory alive in `keep`."""
    try:                                                     # as it mostly is
        if t.get_device() == index and t.dtype is dtype and t.shape == shape and t.is_contiguous() and not t.is_neg():
            keep.append(t)
            return t.data_ptr()
    except (AttributeError, RuntimeError):
        pass
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == index and t.layout is torch.strided):
        _on_gpu(keep[0], **{name: t})
    if t.dtype != dtype:
        raise TypeError("%s must be %s, not %s" % (name, str(dtype)[6:], t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have the shape %s, not %s" % (name, tuple(shape), tuple(t.shape)))
    if t.is_neg() or not t.is_contiguous():
        t = t.detach().resolve_neg().contiguous()
    keep.append(t)
    return t.data_ptr()


def _wish(name, value, shape, index, keep, dtype=torch.float32):
    """(a value for each row or 0, one for all)"""
    if not isinstance(value, torch.Tensor):
        return 0, value
    if value.dtype is not dtype or value.shape != shape:
        raise ValueError("%s must be a number or %s %s" % (name, str(dtype)[6:], list(shape)))
    return _pointer(name, value, dtype, shape, index, keep), None


def _number(name, value, least=-_MOST, most=_MOST):
    value = float(value)
    if not least <= value <= most:
        raise ValueError("%s must be from %g to %g" % (name, least, most))
    return value


def _lies_over(rows, t):
    """Whether a row of `rows` has memory with `t`, whose elements follow one another, in common."""
    n, cols = rows.shape
    size, begin, long = rows.element_size(), t.data_ptr() - rows.data_ptr(), t.numel() * t.element_size()
    line = rows.stride(0) * size if n > 1 else cols * size
    if not (n and long) or begin + long <= 0 or begin >= (n - 1) * line + cols * size:
        return False
    return not (begin >= 0 and cols * size <= begin % line <= line - long)           # (between two rows)


def adjust_logits(logits, ids=None, offsets=None, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0, bias_ids=None, bias=None, allowed=None,
                  allowed_rows=None, out=None):
    """Logits [n, vocab] (float32, bfloat16 or float16) as the requests that they answer ask for them, in this order:

    penalties    for what has been said: row i's history is ids[offsets[i]:offsets[i + 1]] (int32 or int64 ids, one row's after another's, int32 n + 1 offsets, as
                 `Tokenizer.encode_batch_to_device` gives them).  For ids in it l > 0 becomes l / repetition, others l * repetition; for ids that come `count` times behind the
                 row's first prompt_lengths[i] (int32 [n]; None: all of the history counts), l - frequency * count - presence is next.  Ids outside the vocabulary are left out
    biases       bias_ids int32 and bias float32 [n, k], or [k] for all rows, k up to 1024: added to these ids' logits, all of them where an id comes more than once.  A
                 negative id is no entry
    masks        allowed: int32 [m, ceil(vocab / 32)], or without the m one for all rows; where bit id % 32 of word id // 32 is 0 the logit becomes -inf, whatever it was.  Row i has mask
                 allowed_rows[i] (int32 [n]; negative: none; beyond m: nothing is allowed), or mask i without them

    repetition (above 0), presence, frequency: a number, or float32 [n]; they need `ids`.  out: where to write, `logits` itself included, apart from all other
    arguments; else a new tensor is returned."""
    _no_gradient("adjust_logits", logits, repetition, presence, frequency, bias, out)
    index = _on_gpu(logits, logits=logits)
    _logits_of(logits)
    n, vocab = logits.shape
    per_row, keep = torch.Size((n,)), [logits]
    flat_at = n_ids = bits = offsets_at = prompts_at = rho_at = presence_at = frequency_at = entries = bias_ids_at = bias_at = bias_stride = 0
    allowed_at = rows_at = count = stride = 0
    rho, pres, freq = 1.0, 0.0, 0.0
    if (ids is None) != (offsets is None):
        raise ValueError("ids and offsets go together")
    if ids is not None:
        if ids.dim() != 1:
            raise ValueError("ids must have one dimension")
        _on_gpu(logits, ids=ids)
        flat = _ids_of("ids", ids)
        keep.append(flat)
        flat_at, n_ids, bits = flat.data_ptr(), flat.shape[0], _IDS[flat.dtype]
        offsets_at = _pointer("offsets", offsets, torch.int32, (n + 1,), index, keep)
        if prompt_lengths is not None:
            prompts_at = _pointer("prompt_lengths", prompt_lengths, torch.int32, per_row, index, keep)
        rho_at, one = _wish("repetition", repetition, per_row, index, keep)
        rho = 1.0 if rho_at or one is None else _number("repetition", one, _LEAST)
        presence_at, one = _wish("presence", presence, per_row, index, keep)
        pres = 0.0 if presence_at or one is None else _number("presence", one)
        frequency_at, one = _wish("frequency", frequency, per_row, index, keep)
        freq = 0.0 if frequency_at or one is None else _number("frequency", one)
    elif prompt_lengths is not None:
        raise ValueError("prompt_lengths without ids")
    else:
        for name, value, none in (("repetition", repetition, 1.0), ("presence", presence, 0.0), ("frequency", frequency, 0.0)):
            if isinstance(value, torch.Tensor) or value != none:
                raise ValueError("%s without ids" % name)
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    if bias is not None:
        shape = bias_ids.shape
        if len(shape) not in (1, 2) or (len(shape) == 2 and shape[0] != n) or shape[-1] > MAX_BIASES:
            raise ValueError("bias_ids must be [n, k] or [k] with k up to %d" % MAX_BIASES)
        entries, bias_stride = shape[-1], shape[-1] if len(shape) == 2 else 0
        bias_ids_at, bias_at = _pointer("bias_ids", bias_ids, torch.int32, shape, index, keep), _pointer("bias", bias, torch.float32, shape, index, keep)
    if allowed is not None:
        words, shared = -(-vocab // 32), allowed.dim() == 1
        if shared and allowed_rows is not None:
            raise ValueError("allowed_rows needs masks [m, words]")
        if not shared and (allowed.dim() != 2 or (allowed_rows is None and allowed.shape[0] != n)):
            raise ValueError("allowed must be [m, words] with allowed_rows, [n, words] or [words]")
        allowed_at = _pointer("allowed", allowed, torch.int32, (words,) if shared else (allowed.shape[0], words), index, keep)
        if not allowed_at:                                   # no masks at all: there has to be something that none of them is
            keep.append(torch.empty(1, dtype=torch.int32, device=logits.device))
            allowed_at = keep[-1].data_ptr()
        count, stride = (n, 0) if shared else (allowed.shape[0], words)
        if allowed_rows is not None:
            rows_at = _pointer("allowed_rows", allowed_rows, torch.int32, per_row, index, keep)
    elif allowed_rows is not None:
        raise ValueError("allowed_rows without allowed")
    if out is not None:
        _on_gpu(logits, out=out)
        if out.shape != logits.shape or out.dtype != logits.dtype or (vocab > 1 and out.stride(1) != 1) or (n > 1 and out.stride(0) < vocab) or out.is_neg():
            raise ValueError("out must have the logits' shape and type, the elements of a row next to one another and rows apart, and be no view of negated ones")
        # (what one row or one column is apart from the next says nothing)
        same = (out.data_ptr() == logits.data_ptr() and (n < 2 or out.stride(0) == logits.stride(0)) and (vocab < 2 or out.stride(1) == logits.stride(1)) and not logits.is_neg())
        if not same and _overlap(_rows(logits), out):
            raise ValueError("out and logits overlap")
        for t in keep[1:]:                                   # (blocks would read what others have written)
            if _lies_over(out, t):
                raise ValueError("out overlaps another argument")
    result = _there(index, _adjust, logits, out, index, keep, (flat_at, n_ids, bits, entries, offsets_at, prompts_at, rho_at, presence_at, frequency_at, rho, pres, freq, 0,
                                                              bias_ids_at, bias_at, bias_stride, allowed_at, rows_at, count, stride))
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return result


def _adjust(logits, out, index, keep, rest):
    rows = _rows(logits)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    if logits.shape[0]:
        memory = bytearray(ctypes.sizeof(_Adjustment))
        _ADJUSTMENT.pack_into(memory, 0, *_parts(rows), *_parts(out), *rest, _stream(index))
        code = _lib().gtok_x_adjust_logits(_Adjustment.from_buffer(memory))
        if code:
            _done(code, "gtok_x_adjust_logits")
    return out


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(ids int32 [n], logprobs float32 [n]): an id for each row of logits [n, vocab] (float32, bfloat16 or float16).

    u: random numbers, float32 or float64 [n], from 0 and below 1.  With m = exp((l - max) / temperature), ids go in order of falling logits, equal ones in order of rising ids.
    Kept are the first top_k (0: all); of these the fewest whose m make up at least top_p of theirs (1: all); of these the ones with m >= min_p (0: all); the first one in any
    case.  The id is the first one, in the order of ids, at which the running sum of the kept m exceeds u times their sum.  logprobs: the logarithm of its share of all m, kept or not.
    Temperature 0: the first id in that order, logprob 0.

    temperature, top_p, min_p: a number, or float32 [n]; top_k: a number, or int32 [n].  Where the cuts lie and which id is hit is decided by
    whole numbers of up to 50 bits in place of the m, off by no more than 2^-43 relative and, all of a row's together, 2^-25 of their sum.  A row of -inf only gives
    id -1 and logprob -inf; a row with a NaN, or one of a tensor's values that makes no sense (a negative temperature, a `u` of 1), gives id -1 and logprob NaN."""
    _no_gradient("sample", logits, u, temperature, top_p, min_p)
    index = _on_gpu(logits, logits=logits, u=u)
    _logits_of(logits)
    shape, keep = logits.shape[:1], [logits]
    if u.shape != shape or (u.dtype != torch.float32 and u.dtype != torch.float64):
        raise ValueError("u must be float32 or float64 [%d]" % shape[0])
    u_at = _pointer("u", u, u.dtype, shape, index, keep)
    heat_at, heat = _wish("temperature", temperature, shape, index, keep)
    k_at, k = _wish("top_k", top_k, shape, index, keep, torch.int32)
    p_at, p = _wish("top_p", top_p, shape, index, keep)
    least_at, least = _wish("min_p", min_p, shape, index, keep)
    heat = 0.0 if heat is None else _number("temperature", heat, 0.0)
    k = 0 if k is None else min(max(int(k), 0), 1 << 30)
    p = 0.0 if p is None else _number("top_p", p)
    least = 0.0 if least is None else _number("min_p", least)
    return _there(index, _sample, logits, index, keep, (u_at, 64 if u.dtype == torch.float64 else 32, k, heat_at, k_at, p_at, least_at, heat, p, least, 0))


def _sample(logits, index, keep, rest):
    rows = _rows(logits)
    n = rows.shape[0]
    ids = torch.empty(n, dtype=torch.int32, device=logits.device)
    logprobs = torch.empty(n, dtype=torch.float32, device=logits.device)
    if n:
        memory = bytearray(ctypes.sizeof(_Draw))
        _DRAW.pack_into(memory, 0, *_parts(rows), *rest, ids.data_ptr(), logprobs.data_ptr(), _stream(index))
        code = _lib().gtok_x_sample(_Draw.from_buffer(memory))
        if code:
            _done(code, "gtok_x_sample")
    return ids, logprobs
