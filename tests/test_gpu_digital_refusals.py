"""Arguments of the digital operators that no number or truth value can be made of, or one beyond all ranges."""
import pytest
import torch

from aihwkit_amd import _cabi, digital

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("general", [False, True], ids=["native", "general"])
def test_numbers_of_adapters_beyond_all_ranges(general, monkeypatch):
    if general:
        monkeypatch.setattr(_cabi, "_torch_calls", _cabi._GeneralPath())
    index = torch.zeros(80, dtype=torch.int32, device="cuda")
    for n in (1 << 70, -(1 << 70), 1 << 63, 1 << 40, 65536, 0, -1):
        with pytest.raises(RuntimeError, match="number of adapters"):
            digital.AdapterRows(index, n)
    assert digital.AdapterRows(index, 1).rows == 80


def test_flags_without_a_truth_value():
    x, index, flag = torch.zeros(80, 8, device="cuda"), torch.zeros(80, dtype=torch.int32, device="cuda"), torch.zeros(3, device="cuda")
    adapters = digital.LowRankAdapters(torch.zeros(1, 2, 8, device="cuda"), torch.zeros(1, 8, 2, device="cuda"))
    for call in (lambda: digital.dropout(x, 0.5, 1, non_blocking=flag), lambda: digital.layer_norm(x, non_blocking=flag),
                 lambda: adapters.forward(x, index, non_blocking=flag), lambda: adapters.forward(x, index, return_hidden=flag)):
        with pytest.raises(RuntimeError, match="[Bb]oolean"):
            call()
    assert (digital.dropout(x, 0.5, 1) == 0).all()
