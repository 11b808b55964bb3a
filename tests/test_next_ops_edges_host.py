"""Refusals of the operators from hidden states to ids that need no GPU: they come before anything is looked for on one."""
import ctypes
import os
import subprocess

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture(scope="module")
def ops(built):
    from graphtok_b200 import next_ops
    return next_ops


def calls_with(ops):
    """Each call that could pass a gradient on to what it is given, by the argument's name."""
    logits, u, ids, offsets = torch.zeros(2, 5), torch.zeros(2), torch.zeros(4, dtype=torch.int32), torch.tensor([0, 2, 4], dtype=torch.int32)
    for name in ("repetition", "presence", "frequency"):
        yield name, lambda t, name=name: ops.adjust_logits(logits, ids, offsets, **{name: t})
    for name in ("temperature", "top_p", "min_p"):
        yield name, lambda t, name=name: ops.sample(logits, u, **{name: t})
    yield "u", lambda t: ops.sample(logits, t)


def test_gradients_of_penalties_and_wishes_are_refused(ops):
    """A learned penalty or temperature would be trained with nothing, and nobody told."""
    for name, call in calls_with(ops):
        leaf = torch.ones(2, requires_grad=True)
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(leaf)
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(leaf * 0.5)
        for fine in (leaf.detach(), torch.ones(2)):
            with pytest.raises(ValueError, match="must be on the GPU"):
                call(fine)
        with torch.no_grad(), pytest.raises(ValueError, match="must be on the GPU"):
            call(leaf)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(torch.ones(2), torch.ones(2)))


def test_penalties_without_a_history_are_refused(ops, monkeypatch):
    """They would change nothing, whatever they say.  (The checks behind the GPU's are reached as on one.)"""
    monkeypatch.setattr(ops, "_on_gpu", lambda first, **others: 0)
    monkeypatch.setattr(ops, "_there", lambda index, f, *args: args[-1])
    logits = torch.zeros(2, 5)
    for name, none in (("repetition", 1.0), ("presence", 0.0), ("frequency", 0.0)):
        for value in (1.2, -1.0, float("nan"), float("inf"), torch.ones(2), torch.ones(3)):
            with pytest.raises(ValueError, match=name + " without ids"):
                ops.adjust_logits(logits, **{name: value})
        assert ops.adjust_logits(logits, **{name: none}) and ops.adjust_logits(logits, **{name: int(none)})
    with pytest.raises(ValueError, match="prompt_lengths without ids"):
        ops.adjust_logits(logits, prompt_lengths=torch.zeros(2, dtype=torch.int32))


def test_what_lies_over_an_output(ops):
    """Against the bytes themselves: every place and length of a list before, in, between and behind the rows of a matrix."""
    room = torch.zeros(120, dtype=torch.uint8)
    for n, cols, line in ((1, 10, 10), (1, 10, 30), (3, 10, 10), (3, 10, 17), (2, 4, 30), (0, 5, 5), (2, 1, 1)):
        rows = room[20:20 + max(n - 1, 0) * line + cols].as_strided((n, cols), (line, 1), 20)
        taken = {20 + r * line + c for r in range(n) for c in range(cols)}
        for begin in range(90):
            for long in (0, 1, 2, 6, 7, 8, 25):
                assert ops._lies_over(rows, room[begin:begin + long]) == bool(taken & set(range(begin, begin + long))), (n, cols, line, begin, long)
    wide = torch.zeros(40, dtype=torch.int64)
    assert ops._lies_over(room[:64].view(torch.float32).view(2, 8), room[60:]) and not ops._lies_over(room[:64].view(torch.float32).view(2, 8), room[64:])
    assert ops._lies_over(wide.view(torch.float32).view(2, 40), wide[39:]) and not ops._lies_over(wide[:20].view(torch.float32).view(2, 20), wide[20:])


def test_an_output_over_another_argument_is_refused(ops, monkeypatch):
    monkeypatch.setattr(ops, "_on_gpu", lambda first, **others: -1)          # (tensors of the host say that they are on GPU -1)
    monkeypatch.setattr(ops, "_there", lambda index, f, *args: args[1])
    room = torch.zeros(400)
    out, behind = room[:120].view(6, 20), room[120:]
    logits = torch.zeros(6, 20)
    ints = lambda t, *shape: t[:torch.Size(shape).numel()].view(torch.int32).view(shape)          # noqa: E731
    for at in (room, room[100:], room[119:]):
        for named in (dict(ids=ints(at, 4), offsets=torch.zeros(7, dtype=torch.int32)), dict(ids=torch.zeros(4, dtype=torch.int32), offsets=ints(at, 7)), dict(bias=at[:12].view(6, 2), bias_ids=torch.zeros(6, 2).int()),
                      dict(bias=torch.zeros(6, 2), bias_ids=ints(at, 6, 2)), dict(allowed=ints(at, 6, 1)), dict(allowed=torch.zeros(2, 1).int(), allowed_rows=ints(at, 6)),
                      dict(ids=torch.zeros(4, dtype=torch.int32), offsets=torch.zeros(7, dtype=torch.int32), repetition=at[:6])):
            with pytest.raises(ValueError, match="overlaps another argument"):
                ops.adjust_logits(logits, out=out, **named)
    assert ops.adjust_logits(logits, out=out, bias=behind[:12].view(6, 2), bias_ids=ints(behind[12:], 6, 2)) is out


def test_one_row_is_its_own_memory_whatever_its_stride_says(ops, monkeypatch):
    monkeypatch.setattr(ops, "_on_gpu", lambda first, **others: -1)
    monkeypatch.setattr(ops, "_there", lambda index, f, *args: args[1])
    room = torch.zeros(3, 4, 5)
    for logits, out in ((room[:1, 0], room[0, :1]), (room[0, :1], room[:1, 0]), (room[:, :1, 0], room[:, 0, :1]), (room[:0, 0], room[:0, 0])):
        assert logits.shape == out.shape and ops.adjust_logits(logits, out=out) is out
    for logits, out in ((room[:2, 0], room[0, :2]), (room[:1, 0], room.view(-1)[1:6].view(1, 5))):
        with pytest.raises(ValueError, match="overlap"):
            ops.adjust_logits(logits, out=out)


@pytest.mark.parametrize("dtype,zeros", [(torch.bfloat16, False), (torch.float16, True)])
def test_tables_are_loaded_as_tensors_are(ops, tmp_path, dtype, zeros):
    """By torch.load as it is called, beside tensors; and not of another size than theirs."""
    import pickle
    table = ops.QuantizedTable(40, 100, 32, dtype, zeros, "cpu")
    table.data.copy_(torch.randint(0, 256, table.data.shape, generator=torch.Generator().manual_seed(1), dtype=torch.uint8))
    torch.save({"out": table, "in": torch.ones(3)}, tmp_path / "model")
    for named in ({}, dict(map_location="cpu"), dict(weights_only=True), dict(weights_only=False), dict(mmap=True)):
        kept = torch.load(tmp_path / "model", **named)["out"]
        assert isinstance(kept, ops.QuantizedTable) and torch.equal(kept.data, table.data)
        assert (kept.shape, kept.group, kept.dtype, kept.zeros) == (table.shape, 32, dtype, zeros)
    for sizes in ((41, 100, 32), (40, 129, 32), (40, 100, 64), (0, 100, 32), (40, 100, 33)):
        class Wrong(ops.QuantizedTable):
            def __reduce__(self):
                return ops.QuantizedTable, (*sizes, dtype, zeros, None, self.data)
        wrong = Wrong(40, 100, 32, dtype, zeros, None, table.data)
        torch.save(wrong, tmp_path / "wrong")
        if ops._lib().gtok_x_table4_bytes(*sizes, zeros) != table.data.numel():
            with pytest.raises((ValueError, ops.GTokError, pickle.UnpicklingError)):
                torch.load(tmp_path / "wrong")


def places(struct, at=0, head=""):
    """(name, offset, size) of all that is in a ctypes struct, matrices by their parts."""
    for name, kind in struct._fields_:
        field = getattr(struct, name)
        if hasattr(kind, "_fields_"):
            yield from places(kind, at + field.offset, head + name + ".")
        else:
            yield head + name, at + field.offset, field.size


def test_structs_and_packed_structs_are_what_a_c_compiler_makes_of_the_header(ops, tmp_path):
    """Every member's place and size; and each value of a packed struct, which the calls use, is in the member of its turn."""
    from conftest import ROOT
    kinds = {"gtok_x_table4": ops._Table4, "gtok_x_adjustment": ops._Adjustment, "gtok_x_draw": ops._Draw}
    lines = ["printf(\"%s %%zu\\n\", sizeof(%s));" % (c, c) for c in kinds]
    for c, struct in kinds.items():
        lines += ["printf(\"%s %s %%zu %%zu\\n\", offsetof(%s, %s), sizeof(((%s*)0)->%s));" % (c, name, c, name, c, name) for name, _, _ in places(struct)]
    (tmp_path / "sizes.c").write_text('#include <stddef.h>\n#include <stdio.h>\n#include "gtok.h"\nint main(void) {\n%s\nreturn 0;\n}\n' % "\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "sizes"), str(tmp_path / "sizes.c")], check=True)
    said = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines()
    want = ["%s %d" % (c, ctypes.sizeof(struct)) for c, struct in kinds.items()]
    want += ["%s %s %d %d" % (c, *place) for c, struct in kinds.items() for place in places(struct)]
    assert said == want
    for packed, struct in ((ops._ADJUSTMENT, ops._Adjustment), (ops._DRAW, ops._Draw)):
        names = [name for name, _, _ in places(struct)]
        memory = bytearray(ctypes.sizeof(struct))
        assert packed.size == len(memory)
        packed.pack_into(memory, 0, *range(1, len(names) + 1))
        got = struct.from_buffer(memory)
        for i, name in enumerate(names):
            value = got
            for part in name.split("."):
                value = getattr(value, part)
            assert value == i + 1, name
