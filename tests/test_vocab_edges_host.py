"""What the vocabulary operators refuse, and what they say about memory and sources, without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from test_vocab_ops_host import loss_args, ops     # noqa: F401  (ops is a fixture)


def test_forward_mode_is_refused(ops):  # noqa: F811
    """A result without a tangent would be taken for a constant."""
    ids = torch.zeros(3, dtype=torch.int32)
    table, rows = torch.zeros(5, 8), torch.zeros(3, 8)
    hidden, weight, lse = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(3)
    teacher, logits = ids[:, None], torch.zeros(3, 1)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.embed(ids, dual(table)), lambda: ops.embed_grad(ids, dual(rows), 5), lambda: ops.embed_grad(ids, rows, 5, out=dual(table)),
                     lambda: ops.cross_entropy(dual(hidden), weight, ids), lambda: ops.cross_entropy(hidden, dual(weight), ids),
                     lambda: ops.cross_entropy_forward(dual(hidden), weight, ids), lambda: ops.cross_entropy_grad(hidden, dual(weight), ids, lse, lse),
                     lambda: ops.cross_entropy_grad(hidden, weight, ids, lse, dual(lse)), lambda: ops.cross_entropy_grad(hidden, weight, ids, dual(lse), lse),
                     lambda: ops.distill(dual(hidden), weight, teacher, logits), lambda: ops.distill(hidden, dual(weight), teacher, logits),
                     lambda: ops.distill_forward(hidden, dual(weight), teacher, logits), lambda: ops.distill_grad(dual(hidden), weight, teacher, logits, lse, lse)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="must be on the GPU"):          # a level without dual tensors is no reason
            ops.embed(ids, table)


@pytest.mark.parametrize("temperature", [3e-39, 4.2e-39, 1.1e-38])
def test_temperatures_below_the_normal_numbers_are_refused(ops, temperature):  # noqa: F811
    """log2(e) / T has to be a number of fp32: at 4.2e-39 1 / T still is and it is not."""
    assert ops._lib().gtok_x_vocab_loss_workspace(loss_args(ops, temperature=temperature), 0) == -1
    assert b"temperature" in ops._lib().gtok_x_last_error()
    assert ops._lib().gtok_x_vocab_loss_workspace(loss_args(ops, temperature=2.0 ** -126), 0) > 0


@pytest.mark.parametrize("n,vocab,width,entries", [(1, 1, 8, 0), (37, 151665, 2048, 0), (300, 50256, 100, 0), (8192, 128256, 2048, 0), (131072, 151665, 1024, 0), (2048, 151665, 2048, 64)])
def test_memory_of_the_forward_pass(ops, n, vocab, width, entries):  # noqa: F811
    """A copy of the rows, their lists, and a maximum and a sum of each row for every 128 ids: not the logits, a 32nd of them."""
    got = ops._lib().gtok_x_vocab_loss_workspace(loss_args(ops, n, vocab, width, entries), 0)
    rows, k = -(-n // 256) * 256, max(1, entries)
    copies = 2 * (rows + (vocab if width % 8 else 0)) * (-(-width // 8) * 8)
    sums = 8 * rows * max(2 * -(-vocab // 256), 8 * 132)
    assert got <= copies + sums + n * (8 + 20 * k) + 16 * 1024


def test_profiles_are_matched_by_all_that_their_kernels_are_made_of(tmp_path, monkeypatch):
    """A change of any source that a kernel includes, directly or not, changes the hash of its profiles and not the other."""
    import re
    import shutil

    from graphtok_b200 import build
    copy = tmp_path / "csrc"
    shutil.copytree(build.CSRC, copy)
    monkeypatch.setattr(build, "CSRC", str(copy))

    def made_of(name, seen):
        if name not in seen and (copy / name).exists():
            seen.add(name)
            for other in re.findall(r'#include "([^"/]+)"', (copy / name).read_text()):
                made_of(other, seen)
        return seen

    hashes = (build.source_hash, build.vocab_source_hash)
    encode, vocab = set(), set()
    for name in build.SOURCES:
        if name.endswith(".cu"):
            made_of(name, vocab if name.startswith("vocab_") else encode)
    assert "gpu_block.cuh" in encode and "sm100.cuh" in vocab and not encode & vocab
    for names, which in ((encode, 0), (vocab, 1)):
        for name in names:
            before = [h() for h in hashes]
            with open(copy / name, "a") as f:
                f.write("\n")
            after = [h() for h in hashes]
            assert (before[which] != after[which]) and before[1 - which] == after[1 - which], name
