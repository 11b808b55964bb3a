"""What of the vocabulary operators works without a GPU: sizes of workspaces, refusals before anything is queued."""
import ctypes
import math

import pytest
import torch

from graphtok_b200 import GTokError

E = ctypes.c_int32


@pytest.fixture(scope="module")
def ops(built):
    from graphtok_b200 import vocab_ops
    vocab_ops._lib()
    return vocab_ops


def loss_args(ops, n=5, vocab=300, width=64, entries=0, kind=1, temperature=1.0):
    a = ops._Loss()
    a.hidden = ops._Matrix(1 << 20, n, width, width, kind)
    a.weight = ops._Matrix(1 << 20, vocab, width, width, kind)
    a.targets, a.target_bits, a.entries, a.target_stride, a.ignore, a.temperature = 1 << 20, 32, entries, entries, -100, temperature
    if entries:
        a.teacher_logits = ops._Matrix(1 << 20, n, entries, entries, 0)
    return a


def test_workspaces_hold_what_the_passes_keep(ops):
    lib = ops._lib()
    for n, vocab, width, entries in ((1, 1, 1, 0), (37, 151665, 2048, 0), (8192, 128256, 2048, 0), (2048, 151665, 2048, 64), (5, 300, 7, 1024)):
        a = loss_args(ops, n, vocab, width, entries)
        forward, backward = lib.gtok_x_vocab_loss_workspace(a, 0), lib.gtok_x_vocab_loss_workspace(a, 1)
        rows = -(-n // 256) * 256
        k = max(1, entries)
        assert forward >= 2 * rows * width + 12 * n * k + 16 * rows * -(-vocab // 256)
        assert backward >= 2 * rows * width + 8 * n * k + 4 * rows * width
        # never all logits: a piece of dZ is at most 512 MiB, or one tile of the vocabulary
        tables = 2 * (rows + (vocab if width % 8 else 0)) * (width + 8)
        assert backward <= max(512 << 20, 512 * rows) + 4 * (rows * (width + 8) + 8 * 74 * 256 * 256) + tables + 40 * n * k + (1 << 20)
    assert lib.gtok_x_vocab_loss_workspace(loss_args(ops, 0), 0) == 0
    for n, vocab, width in ((0, 5, 3), (1, 1, 1), (2048, 50256, 768), (2049, 300000, 64), (100000, 3, 8192)):
        assert lib.gtok_x_embed_grad_workspace(n, vocab, width) >= 16 * n


@pytest.mark.parametrize("change", [dict(n=-1), dict(vocab=0), dict(width=0), dict(width=1 << 17), dict(entries=1025), dict(entries=-1), dict(kind=0), dict(kind=3),
                                    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan),
                                    dict(temperature=1e-40), dict(n=1 << 31), dict(n=(1 << 28) + 1), dict(vocab=(1 << 30) + 1),
                                    dict(n=1 << 28, vocab=1 << 24)])
def test_sizes_out_of_range_are_refused(ops, change):
    lib = ops._lib()
    assert lib.gtok_x_vocab_loss_workspace(loss_args(ops, **change), 1) == -1
    assert lib.gtok_x_last_error()


def test_lookup_sizes_out_of_range_are_refused(ops):
    lib = ops._lib()
    for n, vocab, width in ((-1, 5, 3), (1, -1, 3), (1, 5, 0), (1 << 31, 5, 3), (1, 1 << 31, 3), (1, 5, (1 << 20) + 1)):
        assert lib.gtok_x_embed_grad_workspace(n, vocab, width) == -1


def test_missing_arguments_are_refused(ops):
    lib = ops._lib()
    assert lib.gtok_x_vocab_loss_workspace(None, 0) == -1
    assert lib.gtok_x_vocab_loss_forward(None) == -1
    assert lib.gtok_x_vocab_loss_backward(None) == -1
    assert lib.gtok_x_embed(None, 32, 1, None, 1.0, None, None) == -1
    assert lib.gtok_x_embed_grad(None, 32, 1, None, 1.0, None, 0, None, 0, None) == -1
    assert lib.gtok_x_next_targets(None, 1, None, 1, None, -100, None, None) == -1


def test_tensors_on_the_host_are_refused(ops):
    ids, table = torch.zeros(3, dtype=torch.int32), torch.zeros(5, 8)
    hidden, weight = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.embed(ids, table), lambda: ops.embed_grad(ids, torch.zeros(3, 8), 5), lambda: ops.next_targets(ids, torch.zeros(2, dtype=torch.int32)),
                 lambda: ops.cross_entropy(hidden, weight, ids), lambda: ops.distill(hidden, weight, ids[:, None], torch.zeros(3, 1))):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()
    for call in (lambda: ops.embed([1, 2], table), lambda: ops.embed(ids, None), lambda: ops.cross_entropy(hidden, weight, [1, 2, 3]),
                 lambda: ops.distill(hidden, weight, ids[:, None], None)):
        with pytest.raises(TypeError, match="must be a torch tensor"):
            call()


def test_without_a_gpu_the_entries_say_so(ops):
    if torch.cuda.is_available():
        pytest.skip("there is a GPU")
    lib = ops._lib()
    assert lib.gtok_x_vocab_loss_forward(loss_args(ops)) == -1 and b"GPU" in lib.gtok_x_last_error()
    with pytest.raises(GTokError, match="no GPU"):
        ops._done(lib.gtok_x_embed(None, 32, 0, None, 1.0, None, None), "gtok_x_embed")
