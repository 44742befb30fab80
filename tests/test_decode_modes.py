"""CPU: operands of the memory recurrence that are not on one CUDA device are refused before a kernel gets their addresses, also
where the autograd function is all that is called (a traced call). The "meta" device stands for another device."""
import pytest
import torch

from atlas_rnn_b200.ops import MemoryRecurrenceFn, Spec, _on_one_device, decode_step


def operands(device="cpu"):
    z = lambda *s: torch.zeros(*s, device=device)
    return [z(2, 1, 8), z(2, 1, 8), z(2, 1, 8), z(2, 1), z(2, 1), z(2, 1), None, z(2, 8, 8), z(2, 8, 8), z(2, 8, 8), None, None]


@pytest.mark.parametrize("call", [MemoryRecurrenceFn.apply, decode_step])
def test_tensors_of_the_host_are_refused(call):
    with pytest.raises(RuntimeError, match="must be on a CUDA device"):
        call(Spec(), *operands())


def test_operands_of_several_devices_are_refused():
    class Cuda:  # a tensor's device, as the check reads it
        device = torch.device("cuda:0")

    _on_one_device(Cuda(), Cuda(), None)
    with pytest.raises(RuntimeError, match="cuda:0 and meta"):
        _on_one_device(Cuda(), None, torch.zeros(1, device="meta"))
    with pytest.raises(RuntimeError, match="cuda:0 and cpu"):
        _on_one_device(Cuda(), torch.zeros(1))
