"""What lx_rotate, lx_causal_conv and lx_linear_attention refuse, and the frequencies of scaled rotations; no call here reaches the device."""

import ctypes
import math

import pytest
import torch

from dromos_amd import abi
from dromos_amd.abi import BF16, F32, Kernels, LxDecay, LxKv8Batch, LxStates, hip_library_path


@pytest.fixture(scope="module")
def lx():
    return Kernels(hip_library_path(), "cpu")  # "cpu": no stream is asked of torch


T4 = torch.zeros(4096, dtype=torch.uint8)
HERE = T4.data_ptr() // 16 * 16 + 16


def batch(seqs=2, rows=HERE, lengths=HERE, max_rows=3):
    return ctypes.pointer(LxKv8Batch(seqs, rows, lengths, None, 0, max_rows, 0))


def states(given=HERE, kept=HERE, slots=None, count=2):
    return ctypes.pointer(LxStates(given, kept, slots, count))


def rotate(lx, **changes):
    a = {"x": HERE, "x_dtype": BF16, "ld_x": 128, "y": HERE, "y_dtype": BF16, "ld_y": 128, "batch": batch(), "positions": None, "freq": HERE, "amplitude": 1.0,
         "rot": 64, "interleaved": 0, "T": 0, "heads": 2, "dim": 64, "stream": None}
    a.update(changes)
    return lx.status("rotate", *a.values())


def conv(lx, **changes):
    a = {"x": HERE, "x_dtype": BF16, "ld_x": 64, "weight": HERE, "bias": None, "w_dtype": BF16, "width": 4, "act": 1, "batch": batch(), "states": states(),
         "y": HERE + 512, "y_dtype": BF16, "ld_y": 64, "T": 0, "C": 64, "stream": None}
    a.update(changes)
    return lx.status("causal_conv", *a.values())


def decay(kind=abi.DECAY_HEAD, x=None, dtype=F32, ld=4, rate=HERE, bias=None):
    return ctypes.pointer(LxDecay(kind, x, dtype, ld, rate, bias))


def linear(lx, **changes):
    a = {"q": HERE, "k": HERE, "v": HERE, "dtype": BF16, "ld_q": 128, "ld_k": 128, "ld_v": 256, "decay": decay(), "skip": None, "gate": None, "gate_dtype": BF16,
         "ld_gate": 256, "batch": batch(), "states": states(), "out": HERE, "out_dtype": BF16, "ld_out": 256, "T": 0, "heads": 4, "k_heads": 2, "dk": 64, "dv": 64,
         "scale": 1.0, "workspace": None, "stream": None}
    a.update(changes)
    return lx.status("linear_attention", *a.values())


def test_calls_without_rows(lx):
    assert rotate(lx) == 0 and conv(lx) == 0 and linear(lx) == 0
    nothing = batch(0, None, None, 0)
    assert rotate(lx, T=5, batch=nothing) == 0 and conv(lx, T=5, batch=nothing) == 0 and linear(lx, T=5, batch=nothing) == 0
    bounded = batch(max_rows=0)  # no sequence has a row that counts
    assert rotate(lx, T=5, batch=bounded) == 0 and conv(lx, T=5, batch=bounded) == 0 and linear(lx, T=5, batch=bounded) == 0
    assert rotate(lx, T=5, heads=0) == 0 and conv(lx, T=5, C=0) == 0


@pytest.mark.parametrize("changes", [
    {"T": -1}, {"T": 1 << 30}, {"batch": None}, {"batch": batch(-1)}, {"batch": batch(max_rows=-1)}, {"heads": -1}, {"dim": -1}, {"dim": 1025}, {"rot": -2},
    {"rot": 7}, {"rot": 66}, {"x_dtype": 2}, {"y_dtype": -1}, {"T": 3, "x": None}, {"T": 3, "y": None}, {"T": 3, "freq": None}, {"T": 3, "ld_x": 127},
    {"T": 3, "ld_y": 127}, {"T": 3, "batch": batch(lengths=None)}, {"T": 3, "y_dtype": F32}, {"T": 3, "ld_y": 256}, {"T": 1 << 29, "heads": 4, "ld_x": 256, "ld_y": 256},
    {"T": -1, "positions": HERE}, {"T": 1 << 30, "positions": HERE}])
def test_rotate_refuses(lx, changes):
    assert rotate(lx, **changes) == 1


@pytest.mark.parametrize("changes", [
    {"T": -1}, {"T": 1 << 30}, {"batch": None}, {"batch": batch(-1)}, {"batch": batch(max_rows=-1)}, {"width": 1}, {"width": 9}, {"C": -1}, {"C": (1 << 24) + 1},
    {"act": 2}, {"x_dtype": 2}, {"w_dtype": 2}, {"y_dtype": 2}, {"states": states(count=-1)}, {"T": 3, "x": None}, {"T": 3, "weight": None}, {"T": 3, "y": None},
    {"T": 3, "y": HERE}, {"T": 3, "ld_x": 63}, {"T": 3, "ld_y": 63}])
def test_conv_refuses(lx, changes):
    assert conv(lx, **changes) == 1


@pytest.mark.parametrize("changes", [
    {"T": -1}, {"T": 1 << 30}, {"batch": None}, {"batch": batch(-1)}, {"batch": batch(max_rows=-1)}, {"heads": 3}, {"heads": 0}, {"k_heads": 0}, {"heads": 4098},
    {"dk": 0}, {"dk": 12}, {"dk": 264}, {"dv": 0}, {"dv": 12}, {"dv": 520}, {"dtype": 2}, {"out_dtype": 2}, {"gate": HERE, "gate_dtype": 2}, {"decay": None},
    {"decay": decay(3)}, {"decay": decay(abi.DECAY_LOG, HERE, 2)}, {"states": states(count=-1)}, {"states": states(given=HERE + 4)}, {"states": states(kept=HERE + 8)},
    {"workspace": HERE + 8}, {"T": 3, "q": None}, {"T": 3, "k": None}, {"T": 3, "v": None}, {"T": 3, "out": None}, {"T": 3, "decay": decay(rate=None)},
    {"T": 3, "decay": decay(abi.DECAY_LOG)}, {"T": 3, "decay": decay(abi.DECAY_STEP)}, {"T": 3, "decay": decay(abi.DECAY_STEP, HERE, F32, 3)}, {"T": 3, "ld_q": 127},
    {"T": 3, "ld_k": 127}, {"T": 3, "ld_v": 255}, {"T": 3, "ld_out": 255}, {"T": 3, "gate": HERE, "ld_gate": 255}])
def test_linear_attention_refuses(lx, changes):
    assert linear(lx, **changes) == 1


def test_workspace_sizes_refuse(lx):
    size = lambda *sizes, b=batch(): lx.size("linear_attention_workspace_bytes", b, *sizes)  # noqa: E731
    assert size(0, 4, 2, 64, 64) == 0
    for bad in ((-1, 4, 2, 64, 64), (1, 4, 3, 64, 64), (1, 4, 2, 60, 64), (1, 4, 2, 64, 516)):
        assert size(*bad) == -1
    assert size(1, 4, 2, 64, 64, b=None) == -1


# ---- the frequencies of scaled rotations ------------------------------------------------------------------------------------


def frequencies(lx, kind, base, rot, factor=1.0, original=4096.0, low=1.0, high=32.0):
    freq, amplitude = (ctypes.c_float * max(1, rot // 2))(), ctypes.c_float()
    status = lx.status("rotary_frequencies", kind, base, rot, factor, original, low, high, ctypes.cast(freq, ctypes.c_void_p), ctypes.addressof(amplitude), stream=False)
    return status, list(freq)[:rot // 2], amplitude.value


def near(got, want):
    # The formula in 64 bits and one rounding to f32: half a step, and a hair for pow's own last bits.
    assert len(got) == len(want)
    for g, w in zip(got, want):
        assert abs(g - w) <= w * 2.0**-24 * 1.001


@pytest.mark.parametrize("rot", [2, 64, 128, 130])
@pytest.mark.parametrize("base", [1e4, 5e5])
def test_plain_linear_and_base(lx, rot, base):
    plain = [base ** (-2 * i / rot) for i in range(rot // 2)]
    status, freq, amplitude = frequencies(lx, abi.ROPE_PLAIN, base, rot)
    assert status == 0 and amplitude == 1.0
    near(freq, plain)
    status, freq, amplitude = frequencies(lx, abi.ROPE_LINEAR, base, rot, 8.0)
    assert status == 0 and amplitude == 1.0
    near(freq, [f / 8.0 for f in plain])
    if rot > 2:
        status, freq, amplitude = frequencies(lx, abi.ROPE_BASE, base, rot, 4.0)
        assert status == 0 and amplitude == 1.0
        near(freq, [(base * 4.0 ** (rot / (rot - 2))) ** (-2 * i / rot) for i in range(rot // 2)])
        near(freq[-1:], [plain[-1] / 4.0])  # the slowest wave is slowed by the factor itself


@pytest.mark.parametrize("rot,base,factor,original", [(128, 1e4, 4.0, 4096.0), (64, 1e4, 40.0, 4096.0), (128, 1e6, 32.0, 8192.0), (32, 1e4, 1.0, 128.0)])
def test_by_parts(lx, rot, base, factor, original):
    status, freq, amplitude = frequencies(lx, abi.ROPE_PARTS, base, rot, factor, original)
    dimension = lambda turns: rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    begin, end = max(math.floor(dimension(32.0)), 0), min(math.ceil(dimension(1.0)), rot - 1)
    want = []
    for i in range(rot // 2):
        slowed = min(1.0, max(0.0, (i - begin) / max(end - begin, 1e-3)))
        f = base ** (-2 * i / rot)
        want.append(f / factor * slowed + f * (1 - slowed))
    assert status == 0 and abs(amplitude - (0.1 * math.log(factor) + 1.0)) < 1e-6
    near(freq, want)


def test_by_waves(lx):
    # Waves that turn four times or more in the original context keep their frequency, those that turn less than once are slowed.
    rot, base, factor, original = 128, 5e5, 8.0, 8192.0
    status, freq, amplitude = frequencies(lx, abi.ROPE_WAVES, base, rot, factor, original, 1.0, 4.0)
    want = []
    for i in range(rot // 2):
        f = base ** (-2 * i / rot)
        length = 2 * math.pi / f
        smooth = (original / length - 1.0) / 3.0
        want.append(f if length < original / 4.0 else f / factor if length > original else (1 - smooth) * f / factor + smooth * f)
    assert status == 0 and amplitude == 1.0
    near(freq, want)


@pytest.mark.parametrize("changes", [
    {"kind": 5}, {"kind": -1}, {"base": 1.0}, {"base": math.nan}, {"base": math.inf}, {"rot": 7}, {"rot": -2}, {"rot": 1026}, {"kind": 1, "factor": 0.5},
    {"kind": 2, "factor": math.nan}, {"kind": 2, "rot": 2, "factor": 2.0}, {"kind": 3, "original": 0.0}, {"kind": 3, "low": 32.0}, {"kind": 4, "low": 0.0}])
def test_frequencies_refuse(lx, changes):
    a = {"kind": 0, "base": 1e4, "rot": 64, "factor": 2.0, "original": 4096.0, "low": 1.0, "high": 32.0}
    a.update(changes)
    assert frequencies(lx, *a.values())[0] == 1


def test_frequencies_alone(lx):
    amplitude = ctypes.c_float()
    assert lx.status("rotary_frequencies", abi.ROPE_PARTS, 1e4, 64, 4.0, 4096.0, 1.0, 32.0, None, ctypes.addressof(amplitude), stream=False) == 0
    assert amplitude.value > 1.0
    assert lx.status("rotary_frequencies", abi.ROPE_PLAIN, 1e4, 0, 1.0, 1.0, 1.0, 2.0, None, None, stream=False) == 0
