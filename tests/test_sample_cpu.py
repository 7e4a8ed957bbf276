"""Sampling without a GPU: the torch form against the 64-bit oracle, and refusals
of the C ABI, which come before anything is launched."""

import ctypes
import os
import re

import pytest
import torch

import nibble_amd
from nibble_amd import _lib
from nibble_amd.sampling import sample, sample_reference
from tests import _sample

TYPES = [torch.float16, torch.bfloat16, torch.float32]


def test_header_and_binding_agree():
    path = os.path.join(os.path.dirname(_lib.__file__), "..", "include", "w4a16_sample.h")
    names = set(re.findall(r"^\w+ (w4a16_\w+)\(", open(path).read(), re.MULTILINE))
    assert names == set(_lib.SAMPLE_SIGNATURES)


@pytest.mark.parametrize("row,settings", _sample.EDGES)
@pytest.mark.parametrize("dtype", TYPES)
def test_edges(row, settings, dtype):
    random = torch.tensor(_sample.EDGE_NUMBERS)
    logits = torch.tensor([row], dtype=dtype).expand(len(random), -1)
    _sample.check(sample(logits, random, **settings), logits, random, **settings)


@pytest.mark.parametrize("settings", [{}, {"top_k": 5}, {"top_p": 0.9}, {"min_p": 0.1}, {"temperature": 0.6, "top_k": 40},
                                      {"temperature": 1.4, "top_k": 300, "top_p": 0.8, "min_p": 0.01}])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows(dtype, settings):
    logits, random = _sample.logits(9, 1003, dtype, 1), _sample.numbers(9, 2)
    _sample.check(sample(logits, random, **settings), logits, random, **settings)


def test_settings_of_rows():
    logits, random = _sample.logits(6, 500, torch.float32, 3), _sample.numbers(6, 4)
    settings = {"temperature": torch.tensor([1.0, 0.0, 0.5, -1.0, 2.0, float("nan")]),
                "top_k": torch.tensor([0, 3, -7, 5, 1, 900]), "top_p": torch.tensor([0.5, 1.0, 2.0, float("nan"), -1.0, 0.9]),
                "min_p": torch.tensor([0.0, -1.0, 0.3, 5.0, float("nan"), 0.1])}
    _sample.check(sample(logits, random, **settings), logits, random, **settings)


def test_tokens_come_as_often_as_they_are_likely():
    """Of N numbers spread evenly a token takes its probability times N, by one more or less."""
    logits = _sample.logits(1, 37, torch.float32, 5)
    count = 4096
    random = (torch.arange(count) + 0.5) / count
    got = torch.bincount(sample(logits.expand(count, -1), random, temperature=0.8), minlength=37)
    share = torch.softmax(logits[0].double() / 0.8, dim=0)
    assert ((got - count * share).abs() <= 1 + 1e-6).all()


def test_refusals_of_the_torch_form():
    logits, random = torch.zeros((2, 5)), torch.zeros(2)
    for error, call in [(TypeError, lambda: sample(logits.double(), random)), (ValueError, lambda: sample(logits[0], random)),
                        (ValueError, lambda: sample(logits, random[:1])), (TypeError, lambda: sample(logits, random.double())),
                        (ValueError, lambda: sample(logits, random, temperature=-1.0)),
                        (ValueError, lambda: sample(logits, random, temperature=float("nan"))),
                        (ValueError, lambda: sample(logits, random, top_k=-1)),
                        (ValueError, lambda: sample(logits, random, top_p=1.5)),
                        (ValueError, lambda: sample(logits, random, min_p=-0.1)),
                        (TypeError, lambda: sample(logits, random, top_k=torch.zeros(2))),
                        (TypeError, lambda: sample(logits, random, top_p=torch.zeros(2, dtype=torch.float64))),
                        (ValueError, lambda: sample(logits, random, min_p=torch.zeros(3))),
                        (ValueError, lambda: sample(logits[:, :0], random)),
                        (ValueError, lambda: sample(logits.clone().requires_grad_(), random))]:
        with pytest.raises(error):
            call()
    assert sample(logits[:0], random[:0]).shape == (0,)
    assert nibble_amd.sample is sample and sample_reference(logits, random).tolist() == [0, 0]


def test_refusals_of_the_c_abi():
    none = _lib.SampleSettings(1.0, 0, 1.0, 0.0, None, None, None, None)

    def call(rows=2, n=100, stride=100, kind=0, logits=1 << 20, random=1 << 21, tokens=1 << 22, settings=none):
        return _lib.lib().w4a16_sample(logits, rows, n, stride, kind, random,
                                       None if settings is None else ctypes.byref(settings), tokens, None)

    of = lambda *values: _lib.SampleSettings(*values, None, None, None, None)  # noqa: E731
    assert call(rows=0) == _lib.W4A16_OK
    assert call(kind=3) == _lib.W4A16_ERR_CONFIG
    assert call(n=0) == call(rows=-1) == _lib.W4A16_ERR_SHAPE
    assert call(n=(1 << 19) + 1) == call(rows=1 << 22) == _lib.W4A16_ERR_TOO_LARGE
    assert call(logits=None) == call(random=None) == call(tokens=None) == call(settings=None) == _lib.W4A16_ERR_NULL
    assert call(logits=(1 << 20) + 1) == call(logits=(1 << 20) + 2, kind=2) == _lib.W4A16_ERR_ALIGNMENT
    for bad in (of(-1.0, 0, 1.0, 0.0), of(float("nan"), 0, 1.0, 0.0), of(1.0, -1, 1.0, 0.0), of(1.0, 0, 1.1, 0.0),
                of(1.0, 0, -0.1, 0.0), of(1.0, 0, 1.0, 1.5), of(1.0, 0, 1.0, float("nan"))):
        assert call(settings=bad) == _lib.W4A16_ERR_CONFIG
