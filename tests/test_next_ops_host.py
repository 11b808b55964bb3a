"""What of the operators from hidden states to ids works without a GPU: sizes of tables, refusals before anything is queued."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture(scope="module")
def ops(built):
    from graphtok_b200 import next_ops
    next_ops._lib()
    return next_ops


@pytest.mark.parametrize("vocab,width,group", [(1, 1, 32), (50256, 768, 64), (128256, 4096, 128), (33, 65, 64), (1000, 8191, 8192), (7, 100, 192)])
def test_a_table_takes_half_a_byte_an_element_and_its_scales(ops, vocab, width, group):
    rows, cols = -(-vocab // 32) * 32, -(-width // 64) * 64
    groups = cols // 32 if group == 32 else -(-width // group)
    for zeros in (0, 1):
        need = rows * cols // 2 + rows * groups * (2 + zeros)
        assert need <= ops._lib().gtok_x_table4_bytes(vocab, width, group, zeros) <= need + 512


@pytest.mark.parametrize("vocab,width,group", [(0, 5, 32), (5, 0, 32), (-1, 5, 32), (5, -1, 32), (5, 5, 0), (5, 5, 16), (5, 5, 33), (5, 5, 96), (5, 5, -64), (5, 5, 1 << 17),
                                               (5, (1 << 16) + 1, 64), ((1 << 24) + 1, 5, 64)])
def test_sizes_out_of_range_are_refused(ops, vocab, width, group):
    assert ops._lib().gtok_x_table4_bytes(vocab, width, group, 0) == -1
    assert ops._lib().gtok_x_last_error()


def test_without_a_gpu_every_entry_says_so(ops):
    if torch.cuda.is_available():
        pytest.skip("there is one")
    lib = ops._lib()
    table, matrix = ops._Table4(), ops._Matrix()
    for call in (lambda: lib.gtok_x_table4_pack(table, None, 0, matrix, None, 0, None), lambda: lib.gtok_x_table4_quantize(table, matrix, None),
                 lambda: lib.gtok_x_table4_logits(matrix, table, matrix, None), lambda: lib.gtok_x_adjust_logits(ops._Adjustment()), lambda: lib.gtok_x_sample(ops._Draw()),
                 lambda: lib.gtok_x_adjust_logits(None), lambda: lib.gtok_x_sample(None)):
        assert call() == -1 and b"GPU" in lib.gtok_x_last_error()


def test_structs_are_the_header_s(ops):
    """Sizes that a C compiler gives the structs of gtok.h."""
    assert ctypes.sizeof(ops._Table4) == 48 and ctypes.sizeof(ops._Adjustment) == 80 + 24 + 40 + 16 + 24 + 40 and ctypes.sizeof(ops._Draw) == 40 + 16 + 32 + 16 + 24


def test_tensors_on_the_host_are_refused(ops):
    logits = torch.zeros(2, 5)
    for call in (lambda: ops.quantize_table(torch.zeros(4, 64)), lambda: ops.pack_table(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 1).half()),
                 lambda: ops.adjust_logits(logits), lambda: ops.sample(logits, torch.zeros(2))):
        with pytest.raises(ValueError, match="must be on the GPU"):
            call()
    with pytest.raises(TypeError, match="QuantizedTable"):
        ops.table_logits(torch.zeros(1, 64).half(), torch.zeros(4, 64).half())
    with pytest.raises(ValueError, match="group"):
        ops.quantize_table(torch.zeros(4, 64), group=48)


def test_gradients_are_refused(ops):
    """A result without the gradient that it should have would be taken for a constant."""
    leaf = torch.zeros(2, 5, requires_grad=True)
    for call in (lambda: ops.adjust_logits(leaf), lambda: ops.sample(leaf, torch.zeros(2)), lambda: ops.adjust_logits(torch.zeros(2, 5), bias=leaf, bias_ids=torch.zeros(2, 5).int())):
        with pytest.raises(NotImplementedError, match="no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="must be on the GPU"):
            call()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(2, 5), torch.ones(2, 5))
        for call in (lambda: ops.adjust_logits(dual), lambda: ops.sample(dual, torch.zeros(2))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
