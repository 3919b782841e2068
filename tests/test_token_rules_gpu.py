"""A request's rules through the step runner and the queue: against the equations on the logits of the same steps without rules."""
import numpy as np
import pytest

import fokonex_reference as ref
import serving_step_reference as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def backend():
    from hologram_b200.backend import B200Backend
    b = B200Backend()
    yield b
    b.close()


@pytest.fixture(scope="module")
def model_dir(tmp_path_factory):
    cfg = ref.CONFIGS["odd"]
    return ref.write_model(tmp_path_factory.mktemp("rules") / "odd", cfg, ref.random_tensors(cfg, seed=4)), cfg


def make_runner(backend, path, **kw):
    from hologram_b200 import decode, models
    return decode.StepRunner(backend, models.load_model(path, "float32"), 64, **kw)


def expect(got, logits, rules, tokens, generated, vocab):
    """f32 logits after the rules: each of seven roundings at most 2^-24 of the largest intermediate value."""
    allowed = None if rules.mask(vocab, generated) is None else np.unpackbits(rules.mask(vocab, generated).view(np.uint8), bitorder="little")[:vocab].astype(bool)
    want, off = plain.rules(logits, list(tokens), (len(tokens) - len(generated), len(tokens)), (rules.repetition, rules.presence, rules.frequency, 0.0), list(rules.bias.items()), allowed)
    # three of the penalties are rounded to f32 on the device, 2^-24 each: ten roundings, less than twice seven
    np.testing.assert_array_equal(np.isneginf(got), np.isneginf(want))
    real = ~np.isneginf(want)
    assert np.all(np.abs(got[real] - want[real]) <= 2 * off[real])


@pytest.mark.parametrize("graphs", [True, False])
def test_rules_of_a_sequence_step_by_step(backend, model_dir, graphs):
    """Prompt portions of one and of several tokens, then single tokens; the second sequence finds nothing of the first."""
    from hologram_b200 import decode
    path, cfg = model_dir
    vocab, rng = cfg["vocab"], np.random.default_rng(3)
    sequences = [(rng.integers(0, vocab, 21), 20, [8, 1, 12]), (rng.integers(0, vocab, 9), 4, [3, 2, 4])]
    rules = [decode.TokenRules(1.3, 0.5, 0.25, {2: 1.5, 5: -np.inf}, allowed=lambda tokens: range(len(tokens) % 3, vocab, 2)), decode.TokenRules(0.7)]
    runner, bare = make_runner(backend, path, graphs=graphs), make_runner(backend, path, graphs=graphs)
    for (tokens, prompt, portions), rule in zip(sequences, rules):
        at = 0
        while at < len(tokens):
            n = portions.pop(0) if portions else 1
            part, at = tokens[at:at + n], at + n
            generated = list(tokens[prompt:at]) if at > prompt else []
            expect(runner.step("a", part, rules=rule, generated=generated)[0], bare.step("a", part)[0], rule, tokens[:at], generated, vocab)
        runner.end("a")
        bare.end("a")
    runner.close()
    bare.close()


def test_a_first_ruled_step_late_in_a_sequence_knows_all_of_it(backend, model_dir):
    from hologram_b200 import decode
    path, cfg = model_dir
    tokens = np.random.default_rng(5).integers(0, cfg["vocab"], 40)
    runner, bare, rule = make_runner(backend, path, max_rows=8), make_runner(backend, path, max_rows=8), decode.TokenRules(1.5, frequency=0.5)
    for r in (runner, bare):
        r.step("a", tokens[:19])
    got, logits = runner.step("a", tokens[19:39], rules=rule, generated=tokens[30:39]), bare.step("a", tokens[19:39])
    expect(got[0], logits[0], rule, tokens[:39], tokens[30:39], cfg["vocab"])
    # without rules again, nothing is left of them
    assert np.array_equal(runner.step("a", tokens[39:]), bare.step("a", tokens[39:]))
    runner.close()
    bare.close()


def test_generation_keeps_to_the_rules(backend, model_dir):
    from hologram_b200 import decode
    path, cfg = model_dir
    runner, prompt = make_runner(backend, path), [3, 1, 4, 1, 5]
    only = decode.generate(runner, prompt, 10, rules=decode.TokenRules(allowed=[7, 11]))
    assert set(only) <= {7, 11}
    # a token once generated is as good as forbidden
    once = decode.generate(runner, prompt, 12, rules=decode.TokenRules(presence=1e9))
    assert len(set(once)) == 12
    sampled = decode.generate(runner, prompt, 12, decode.Sampler(1.0, 0, 3), rules=decode.TokenRules(bias={9: 1e4}))
    assert set(sampled) == {9}
    spelled = decode.generate(runner, prompt, 4, rules=decode.TokenRules(allowed=lambda tokens: [[2], [4], [6], [8]][len(tokens)]))
    assert spelled == [2, 4, 6, 8]
    runner.close()


def test_refused_rules_leave_the_sequence_as_it_was(backend, model_dir):
    from hologram_b200 import decode
    path, cfg = model_dir
    runner = make_runner(backend, path)
    runner.step("a", [1, 2, 3])
    for kw in ({"rules": decode.TokenRules(allowed=[cfg["vocab"]])}, {"rules": decode.TokenRules(bias={cfg["vocab"]: 1.0})}, {"rules": decode.TokenRules(), "want": [0]},
               {"rules": decode.TokenRules(), "want": []}, {"rules": decode.TokenRules(), "generated": [1] * 6}):
        with pytest.raises(ValueError):
            runner.step("a", [4, 5], **kw)
    assert runner.cache.length == 3
    runner.close()
