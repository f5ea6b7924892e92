"""What the operators of beam search refuse, on the CPU: every refusal comes before a launch."""
import pytest
import torch

from pico_vllm_b200 import ops
from pico_vllm_b200.errors import KernelError


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("logits,scores,beams,end,out,match", [
    (torch.zeros(8, 10).double(), torch.zeros(2, 4), 4, None, None, "float32"),
    (torch.zeros(8, 10).bfloat16(), torch.zeros(2, 4), 4, None, None, "float32"),
    (torch.zeros(8, 10), torch.zeros(2, 4).double(), 4, None, None, "float32"),
    (torch.zeros(8), torch.zeros(2, 4), 4, None, None, "logits float32"),
    (torch.zeros(8, 10), torch.zeros(8), 4, None, None, "scores float32"),
    (torch.zeros(7, 10), torch.zeros(2, 4), 4, None, None, "logits float32"),
    (torch.zeros(10, 8).t(), torch.zeros(2, 4), 4, None, None, "contiguous columns"),
    (torch.zeros(8, 10), torch.zeros(4, 2).t(), 4, None, None, "contiguous float32"),
    (torch.zeros(8, 10), torch.zeros(2, 4), 3, None, None, "no more rows than beams"),
    (torch.zeros(8, 10), torch.zeros(2, 4), 33, None, None, "1 to 32 beams"),
    (torch.zeros(0, 10), torch.zeros(2, 0), 4, None, None, "no more rows than beams"),
    (torch.zeros(8, 10), torch.zeros(2, 4), 4, 10, None, "end token"),
    (torch.zeros(8, 10), torch.zeros(2, 4), 4, -1, None, "end token"),
    (torch.zeros(8, 10), torch.zeros(2, 4), 4, None, i32(31), "out must be"),
    (torch.zeros(8, 10), torch.zeros(2, 4), 4, None, torch.zeros(32), "out must be"),
    (torch.zeros(8, 10), torch.zeros(2, 4), 4, 3, None, "CUDA tensors"),
])
def test_choice_refuses(logits, scores, beams, end, out, match):
    with pytest.raises(KernelError, match=match):
        ops.beam_select(logits, scores, beams, end, out)


ROWS = [
    (torch.zeros(2, 3, 4), "a list of tensors"),          # (a list of its entries would be something else)
    ((t for t in [torch.zeros(2, 3, 4)]), "a list of tensors"),
    ([torch.zeros(5)], "entries, rows"),
    ([torch.zeros(2, 3, 4, 5).transpose(2, 3)], "in one piece"),
    ([torch.zeros(2, 3, 4)[:, :, ::2]], "in one piece"),
    ([torch.zeros(1, 1, 4).expand(2, 3, 4)], "overlap"),
    ([torch.zeros(2, 1, 4).expand(2, 3, 4)], "overlap"),
    ([torch.zeros(100).as_strided((2, 3, 4), (6, 4, 1))], "overlap"),
    ([torch.zeros(2, 3, 4)], "CUDA tensors"),
]


@pytest.mark.parametrize("tensors,match", ROWS)
def test_rows_refuse(tensors, match):
    with pytest.raises(KernelError, match=match):
        ops.copy_pages(tensors, i32(3), i32(3))
    with pytest.raises(KernelError, match=match):
        ops.reorder_states(tensors, i32(1, 2), i32(1, 2))


def test_one_tensor_twice_is_refused():
    t = torch.zeros(2, 6, 4)
    for tensors in ([t, t], [t, t[:, 1:]], [t[:, ::2], t[:, 1::2]]):
        with pytest.raises(KernelError, match="overlap"):
            ops.copy_pages(tensors, i32(3), i32(3))
        with pytest.raises(KernelError, match="overlap"):
            ops.reorder_states(tensors, i32(1, 2), i32(1, 2))


@pytest.mark.parametrize("src,dst", [(i32(3), i32(4)), (i32(3).long(), i32(3)), (i32(3), i32(3).long()), (i32(3, 1), i32(3, 1)), (i32(6)[::2], i32(3))])
def test_pairs_refused(src, dst):
    with pytest.raises(KernelError, match="src and dst"):
        ops.copy_pages([torch.zeros(2, 3, 4)], src, dst)


@pytest.mark.parametrize("slots,parents,match", [(i32(3), i32(3), "slots and parents"), (i32(2, 3), i32(2, 2), "slots and parents"),
                                                 (i32(2, 3).long(), i32(2, 3), "slots and parents"), (i32(3, 2).t(), i32(2, 3), "slots and parents"),
                                                 (i32(2, 33), i32(2, 33), "1 to 32 places"), (i32(2, 0), i32(2, 0), "1 to 32 places")])
def test_families_refused(slots, parents, match):
    with pytest.raises(KernelError, match=match):
        ops.reorder_states([torch.zeros(2, 3, 4)], slots, parents)
