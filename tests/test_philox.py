"""The oracle of dropout's random numbers against the generator's published answers, and against the other copies of it here."""
import importlib.util
import os

import numpy as np
import pytest

from philox import philox, words

# counter, key, answer: all zeros, all ones, the digits of pi (no two words alike)
ANSWERS = [((0,) * 4, (0,) * 2, (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
           ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
           ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
            (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]


@pytest.mark.parametrize("counter,key,answer", ANSWERS)
def test_published_answers(counter, key, answer):
    assert tuple(philox(counter, key)) == answer


def test_order_of_the_words():
    """Element i: word i % 4 of the counter (i / 4 in the low words, the offset in the high ones) under the seed, low word first."""
    counter, key, answer = ANSWERS[2]
    block, offset, seed = counter[1] << 32 | counter[0], counter[3] << 32 | counter[2], key[1] << 32 | key[0]
    assert tuple(words(4 * block, 4, seed, offset)) == answer
    assert tuple(words(4 * block + 1, 2, seed, offset)) == answer[1:3]


def test_the_gpu_tests_copy():
    """numpy's copy in the tests of dropout, at words that differ from each other."""
    pytest.importorskip("torch")
    from test_gpu_dropout import words as copy
    for seed, offset in ((0x299f31d0a4093822, 0x0370734413198a2e), (1, 2), ((1 << 64) - 1, 1 << 33)):
        assert np.array_equal(copy(1001, seed, offset), np.array(words(0, 1001, seed, offset), np.uint64))


def test_the_performance_cases_copy():
    torch = pytest.importorskip("torch")
    path = os.path.join(os.path.dirname(__file__), "..", "perf", "more_operators.py")
    spec = importlib.util.spec_from_file_location("more_operators", path)
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    arange = torch.arange
    cases.torch = type("OnTheCpu", (), {"__getattr__": lambda _, name: getattr(torch, name),
                                       "arange": staticmethod(lambda *a, device=None, **k: arange(*a, **k))})()
    for seed, offset in ((0x299f31d0a4093822, 0x0370734413198a2e), (3, 1 << 40)):
        assert cases._philox(seed, offset, 100).reshape(-1).tolist() == words(0, 400, seed, offset)
