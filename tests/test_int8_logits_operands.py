"""What int8.logits refuses of its operands' layout.  CPU only: tensors that say that they are on a device, whose
memory nothing reads, and a launch that fails the test if a call reaches it."""
import pytest
import torch

import syntropy_amd.int8 as I

K, N = 64, 8


class OnDevice:
    """A CPU tensor that answers what a device tensor does."""

    def __init__(self, t):
        self.t = t

    is_cuda, device = True, torch.device("cuda:0")

    def get_device(self):
        return 0

    def __getattr__(self, name):
        return getattr(self.t, name)


class Head:
    k_in, n_out, device, bias = K, N, 0, None


@pytest.fixture
def reached(monkeypatch):
    calls = []
    monkeypatch.setattr(I, "_on_stream", lambda *a: calls.append(a))
    return calls


def test_whole_operands_reach_the_launch(reached):
    for g in (torch.ones(K), torch.ones(2 * K)[K:], torch.ones(1, K)):
        I.logits(Head, OnDevice(g), 1e-5, OnDevice(torch.ones(3, K)), 3)
    assert len(reached) == 3


@pytest.mark.parametrize("g", [torch.ones(1).expand(K), torch.ones(K, 2)[:, 0], torch.ones(K // 8, 16)[:, :8],
                               torch.ones(K + 1), torch.ones(K, dtype=torch.float64)],
                         ids=["expanded", "strided", "two-dimensional", "longer", "F64"])
def test_a_gain_that_is_not_its_values_side_by_side(reached, g):
    with pytest.raises(I.GemvError):
        I.logits(Head, OnDevice(g), 1e-5, OnDevice(torch.ones(3, K)), 3)
    assert not reached


@pytest.mark.parametrize("x", [torch.ones(1, K).expand(3, K), torch.ones(3, 2 * K)[:, :K], torch.ones(2, K),
                               torch.ones(3, K, dtype=torch.bfloat16)], ids=["expanded", "strided", "short", "BF16"])
def test_rows_that_are_not_side_by_side(reached, x):
    with pytest.raises(I.GemvError):
        I.logits(Head, OnDevice(torch.ones(K)), 1e-5, OnDevice(x), 3)
    assert not reached


@pytest.mark.parametrize("y", [torch.ones(3, 2 * N)[:, :N], torch.ones(2, N), torch.ones(3, N, dtype=torch.float16)],
                         ids=["strided", "short", "F16"])
def test_outputs_that_are_not_side_by_side(reached, y):
    with pytest.raises(I.GemvError):
        I.logits(Head, OnDevice(torch.ones(K)), 1e-5, OnDevice(torch.ones(3, K)), 3, y=OnDevice(y))
    assert not reached
