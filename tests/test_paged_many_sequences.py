"""Tables of more sequences than the C entries count."""
import pytest
import torch

from codegendemo_b200.kcg import matmul_op

BF = torch.bfloat16


class _Huge(torch.Tensor):
    """A tensor that says it is on a GPU and has no memory."""
    is_cuda = True


def _meta(*shape, dtype=BF):
    return torch.empty(shape, dtype=dtype, device="meta").as_subclass(_Huge)


@pytest.mark.parametrize("sequences", [2 ** 24 + 1, 2 ** 32 + 1])
@pytest.mark.parametrize("op", ["append_kv", "attention_paged"])
def test_they_are_refused(op, sequences):
    """2^32 + 1 of them are 1 in 32 bits."""
    cache = _meta(4, 2, 16, 128)
    table, lengths, starts = _meta(sequences, 1, dtype=torch.int32), _meta(sequences, dtype=torch.int32), _meta(sequences + 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="sequences"):
        if op == "append_kv":
            matmul_op.append_kv(_meta(3, 2, 128), _meta(3, 2, 128), cache, cache, table, lengths, starts)
        else:
            matmul_op.attention_paged(_meta(3, 8, 128), cache, cache, table, lengths, starts)
