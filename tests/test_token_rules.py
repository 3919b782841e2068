"""A request's rules on its logits, on the CPU: their checks, the masks, what the queue and the command line pass on."""
import argparse

import numpy as np
import pytest

from hologram_b200 import decode as dc
from hologram_b200.__main__ import token_rules


@pytest.mark.parametrize("kw", [{"repetition": 0.0}, {"repetition": -1.0}, {"repetition": float("nan")}, {"repetition": float("inf")}, {"presence": float("nan")},
                                {"frequency": float("inf")}, {"bias": {-1: 1.0}}, {"bias": {1: float("nan")}}, {"bias": {1: float("inf")}}, {"allowed": []}, {"allowed": [3, -1]}])
def test_rules_without_sense_are_refused(kw):
    with pytest.raises(ValueError):
        dc.TokenRules(**kw)


@pytest.mark.parametrize("kw", [{"repetition": 1e-46}, {"repetition": 1e39}, {"presence": 1e39}, {"presence": -1e39}, {"frequency": 1e39}, {"bias": {1: 1e39}}, {"bias": {1: -1e39}}])
def test_rules_whose_values_f32_does_not_hold_are_refused(kw):
    with pytest.raises(ValueError):
        dc.TokenRules(**kw)


def test_rules_whose_values_f32_just_holds():
    r = dc.TokenRules(1e-38, 3e38, -3e38, {0: 3e38, 1: -3e38, 2: -float("inf"), 3: 1e-60})
    assert (r.repetition, r.presence, r.frequency, r.bias[0], r.bias[2]) == (1e-38, 3e38, -3e38, 3e38, -float("inf"))


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 64, 100])
def test_masks_have_a_bit_for_each_allowed_token(vocab):
    ids = sorted({0, vocab - 1, vocab // 2})
    words = dc.TokenRules(allowed=ids).mask(vocab, [])
    assert words.dtype == np.uint32 and words.size == (vocab + 31) // 32
    assert [t for t in range(32 * words.size) if words[t // 32] >> (t % 32) & 1] == ids
    assert dc.TokenRules().mask(vocab, []) is None and dc.TokenRules(allowed=lambda tokens: None).mask(vocab, []) is None
    with pytest.raises(ValueError):
        dc.TokenRules(allowed=[vocab]).mask(vocab, [])
    with pytest.raises(ValueError):
        dc.TokenRules(allowed=lambda tokens: []).mask(vocab, [])


def test_rules_that_leave_no_token_are_refused():
    """A step would end with logits of -inf alone, of which a sampler takes a forbidden token."""
    never = -float("inf")
    with pytest.raises(ValueError):
        dc.TokenRules(bias={3: never}, allowed=[3, 3]).mask(8, [])
    with pytest.raises(ValueError):
        dc.TokenRules(bias={0: never, 1: never, 2: 1.0}, allowed=lambda tokens: {0, 1}).mask(8, [])
    with pytest.raises(ValueError):
        dc.TokenRules(bias={0: never, 1: never}).mask(2, [])
    assert dc.TokenRules(bias={3: never}, allowed=[3, 4]).mask(8, [])[0] == 0b11000
    assert dc.TokenRules(bias={0: never}).mask(2, []) is None


def test_an_allowing_function_sees_the_generated_tokens():
    rules = dc.TokenRules(allowed=lambda tokens: [len(tokens)])
    assert rules.mask(8, [])[0] == 1 and rules.mask(8, [5, 5, 6])[0] == 8


class RecordingRunner:
    """Always likes token 1 best; records the rules that its steps are given."""

    def __init__(self, capacity=32, max_rows=4):
        self.cache, self.max_rows, self.calls = dc.SequenceCache(capacity), max_rows, []

    def step(self, seq, tokens, want=None, rules=None, generated=()):
        self.cache.acquire(seq)
        self.calls.append((len(tokens), want, rules, list(generated)))
        return np.array([[0.0, 1.0]], dtype=np.float32)

    def end(self, seq):
        self.cache.release(seq)


def test_the_queue_gives_the_rules_to_the_steps_that_choose_a_token():
    rules, runner = dc.TokenRules(1.5), RecordingRunner()
    assert dc.generate(runner, [0] * 6, 3, rules=rules) == [1, 1, 1]
    assert runner.calls == [(4, [], None, []), (2, None, rules, []), (1, None, rules, [1]), (1, None, rules, [1, 1])]
    runner = RecordingRunner()
    dc.generate(runner, [0] * 6, 2)
    assert [c[2] for c in runner.calls] == [None, None, None]


def test_the_command_line_builds_rules():
    none = dict(repetition=1.0, presence=0.0, frequency=0.0, bias=[], allow=None)
    make = lambda **kw: token_rules(argparse.Namespace(**{**none, **kw}))
    assert make() is None
    r = make(repetition=1.25, presence=0.5, frequency=0.25, bias=["3=-1.5", "7=2"], allow="1,3,7")
    assert (r.repetition, r.presence, r.frequency, r.bias, list(r.allowed)) == (1.25, 0.5, 0.25, {3: -1.5, 7: 2.0}, [1, 3, 7])
    assert make(allow="4").repetition == 1.0 and make(bias=["0=1"]).bias == {0: 1.0}
    with pytest.raises(ValueError):
        make(repetition=0.0)
