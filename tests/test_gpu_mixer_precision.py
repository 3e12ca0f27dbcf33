"""What lx_linear_attention keeps of f32 where little things add up."""

import math

import pytest
import torch

from dromos_amd.abi import BF16, DECAY_HEAD, F32, LxDecay, LxKv8Batch, LxStates
from mixer import pointer

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class Fading:
    """Calls of `rows` rows whose keys are zero: a state of 64 x 64 that only fades, by a constant rate."""

    def __init__(self, hip, rows, rate, seed):
        self.hip, self.rows = hip, rows
        self.before = torch.rand(64, 64, generator=torch.Generator().manual_seed(seed)) + 0.5
        self.state, self.rate = self.before.cuda().view(1, 1, 64, 64), torch.tensor([rate], device="cuda")
        self.x, self.out = torch.zeros(rows, 64, dtype=BF, device="cuda"), torch.empty(rows, 64, dtype=BF, device="cuda")
        self.first = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
        self.decay = LxDecay(DECAY_HEAD, None, F32, 1, self.rate.data_ptr(), None)
        self.batch, self.states = LxKv8Batch(1, self.first.data_ptr(), None, None, 0, rows, 0), LxStates(self.state.data_ptr(), self.state.data_ptr(), None, 1)
        need = int(hip.size("linear_attention_workspace_bytes", pointer(self.batch), rows, 1, 1, 64, 64))
        self.workspace = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")

    def call(self):
        assert self.hip.status("linear_attention", self.x, self.x, self.x, BF16, 64, 64, 64, pointer(self.decay), None, None, BF16, 0, pointer(self.batch),
                               pointer(self.states), self.out, BF16, 64, self.rows, 1, 1, 64, 64, 0.125, self.workspace) == 0

    def errors(self, tokens):
        """The relative errors of the state's values."""
        want = self.before.double() * torch.exp(tokens * self.rate.double().cpu())
        return self.state[0, 0].double().cpu() / want - 1


@pytest.mark.parametrize("rate", [-1e-5, -1e-6])
@pytest.mark.parametrize("rows", [300, 131072])
def test_slow_decays_of_a_prompt(hip, rows, rate):
    """Up to 512 parts, a rounding of half a step, 2^-24, a part: at random 2^-24 sqrt(512 / 3) = 2^-20.3 of a value, and of 4096 values' mean a 64th of that, 2^-26.3,
    four times which is 2^-24.3. To one side: of each part's logarithm 2^-22 (its sum's rounding, the exponential's and a logarithm's), 2^-22 |n rate| together; a sum's
    last place, 2^-40 a token at most, 2^-23 of 131072 of them."""
    f = Fading(hip, rows, rate, 1)
    f.call()
    errors = f.errors(rows)
    assert abs(errors.mean().item()) <= 2.0**-22 * abs(rows * rate) + 2.0**-23
    assert errors.abs().max().item() <= 2.0**-22 * abs(rows * rate) + 2.0**-18


@pytest.mark.parametrize("rows,pieces", [(1, [1]), (6, [1] * 6), (7, [7]), (8, [8]), (64, [64]), (130, [128, 2])])
def test_slow_decays_of_many_short_calls(hip, rows, pieces):
    """8192 calls; a state is rounded once a piece. That is nothing random where a state falls by few steps at a time (6 rows: 4e-6 of a value, to one side), so what is
    compared with is the same in 64 bits rounded as often. Beside that the logarithms' errors, 2^-22 of them as in a prompt, and their last places, 2^-21 of all tokens."""
    calls, whole = 8192, -0.57
    f = Fading(hip, rows, whole / (calls * rows), 2)
    for _ in range(calls):
        f.call()
    rate, state = f.rate.double().item(), f.before.clone()
    fades = [math.exp(rate * n) for n in pieces]
    for _ in range(calls):
        for fade in fades:
            state = (state.double() * fade).float()
    apart = f.state[0, 0].double().cpu() / state.double() - 1
    assert abs(apart.mean().item()) <= 2.0**-22 * -whole + 2.0**-21
    assert apart.abs().max().item() <= 2.0**-22 * -whole + 2.0**-19
