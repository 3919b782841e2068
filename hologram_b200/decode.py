"""Serving a decoder model: the step function over its `.holo` archives, the cache, sampling and the request queue.

A model's archives are fixed step shapes; `StepRunner` keeps one session per row count in use (powers of two, the
portion is padded up) and one per logit count. All of them share the first session's device copies of the weights
and its cache, state, residual stream and position buffers, and replay as CUDA graphs after their first walk. Padding rows
lie after the portion's last token: no real row sees them. What they leave in a plain cache is dropped past its end or
overwritten by a later step before any row can see it; ring caches and recurrent states take the real rows only, by the
row count every step carries, and a state starts from zero where the step's position is 0.
"""
from collections import deque

import numpy as np

from . import kernel_call as kc
from .backend import DeviceWorkspace
from .session import InferenceSession


class CacheFull(RuntimeError):
    """A step or a request needs more positions than the cache has, or the cache belongs to another sequence."""


def bucket(n):
    """The step shape for n rows: the next power of two."""
    b = 1
    while b < n:
        b *= 2
    return b


class SequenceCache:
    """The positions one sequence at a time holds in the sessions' shared cache and state buffers."""

    def __init__(self, capacity):
        self.capacity = capacity
        self.owner, self.length = None, 0

    def acquire(self, owner):
        if self.owner is not None and self.owner != owner:
            raise CacheFull(f"the cache is held by sequence {self.owner!r}")
        if self.owner is None:
            self.owner, self.length = owner, 0

    def check(self, n):
        if self.length + n > self.capacity:
            raise CacheFull(f"{self.length} + {n} positions exceed the cache's {self.capacity}")

    def release(self, owner):
        if self.owner == owner:
            self.owner, self.length = None, 0


class TokenRules:
    """What a request does to its logits before a token is chosen: `repetition` divides positive logits of tokens that the sequence
    has (and multiplies negative ones); `presence` and `frequency` are taken off once, and once for each time, where a token was
    generated; `bias` maps tokens to values added; `allowed` are the only tokens that may come next, as ids or as a function of the
    tokens generated so far that returns ids (None: all). They run on the device as one LogitRules call."""

    def __init__(self, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
        self.repetition, self.presence, self.frequency = float(repetition), float(presence), float(frequency)
        self.bias = {int(t): float(v) for t, v in dict(bias or {}).items()}
        # as the device has them, in f32: what is positive or finite here may not be there
        with np.errstate(over="ignore"):
            repetition, presence, frequency, *values = np.array([self.repetition, self.presence, self.frequency, *self.bias.values()]).astype(np.float32)
        if not (0.0 < repetition < np.inf and np.isfinite(presence) and np.isfinite(frequency)):
            raise ValueError("repetition is positive; repetition, presence and frequency are finite, in f32")
        if any(t < 0 for t in self.bias) or any(np.isnan(v) or v == np.inf for v in values) or any(v == -np.inf and np.isfinite(b) for v, b in zip(values, self.bias.values())):
            raise ValueError("a bias has a token id from 0 on and a value that is finite in f32, or -inf")
        self.allowed = allowed if allowed is None or callable(allowed) else self._ids(allowed)

    @staticmethod
    def _ids(ids):
        ids = np.asarray(list(ids), dtype=np.int64)
        if ids.size == 0 or ids.min() < 0:
            raise ValueError("the allowed tokens are one id at least, from 0 on")
        return ids

    def mask(self, vocab, generated):
        """The allowed tokens as bits of u32 words, or None where all are."""
        ids = self.allowed(list(generated)) if callable(self.allowed) else self.allowed
        banned = {t for t, v in self.bias.items() if v == -np.inf}
        if ids is None:
            if len(banned) >= vocab:
                raise ValueError("the biases leave no token")
            return None
        ids = self._ids(ids)
        if ids.max() >= vocab:
            raise ValueError("an allowed token lies outside the vocabulary")
        if banned and banned.issuperset(ids.tolist()):
            raise ValueError("the biases leave none of the allowed tokens")
        bits = np.zeros((vocab + 31) // 32 * 32, dtype=np.uint8)
        bits[ids] = 1
        return np.packbits(bits, bitorder="little").view(np.uint32)


class StepRunner:
    """Runs portions of a sequence: `step(id, tokens, want)` appends the tokens and returns the logits at the wanted places."""

    LOGIT_ROWS = 256

    def __init__(self, backend, model, capacity, max_rows=2048, graphs=True):
        self.backend, self.model, self.graphs = backend, model, graphs
        self.cache = SequenceCache(capacity)
        self.max_rows = 1
        while self.max_rows < min(max_rows, capacity):
            self.max_rows *= 2
        self._steps, self._heads = {}, {}
        # the single-token step holds every weight: the other shapes borrow from it
        self._root = InferenceSession(backend, model.build_step(1, capacity, self.max_rows, True), verify=False)
        self._steps[1] = [self._root, False]
        # the sequence's tokens, how many of them the device has, and the operands of its rules
        self._tokens, self._sent = np.zeros(capacity, dtype=np.int32), 0
        self._rules_ws, self._rules_bytes = None, 0

    def close(self):
        for table in (self._heads, self._steps):
            for n, (s, _) in list(table.items()):
                if s is not self._root:
                    s.close()
        if self._rules_ws is not None:
            self._rules_ws.close()
            self._rules_ws = None
        self._root.close()
        self._steps, self._heads = {}, {}

    def _session(self, table, rows, build):
        if rows not in table:
            table[rows] = [InferenceSession(self.backend, build(), verify=False, donor=self._root), False]
        return table[rows]

    def _execute(self, entry):
        session, captured = entry
        session.execute()
        if self.graphs and not captured:       # the first walk allocated what it needs: later ones replay it
            session.capture()
            entry[1] = True
        return session

    def _apply(self, session, rules, mask, generated, total):
        """`rules` on the one row of the session's logits, in place."""
        vocab, n = self.model.config.vocab, len(rules.bias)
        if self._rules_ws is None:
            self._rules_ws, self._rules_bytes, self._sent = DeviceWorkspace(self.backend, 3), 0, 0
            self._rules_ws.alloc(1, 4 * self._tokens.size)
        ws = self._rules_ws
        ws.bind(0, *session.device_ptr("logits"))
        if self._sent < total:
            ws.write(kc.rb(1, 4 * self._sent, 4 * (total - self._sent)), self._tokens[self._sent:total])
            self._sent = total
        # spans, params, where the biases begin and end, their tokens, their values, the mask, at multiples of 16 bytes
        words = [np.array([total - len(generated), total], dtype=np.int32), np.array([rules.repetition, rules.presence, rules.frequency, 0.0], dtype=np.float32),
                 np.array([0, n], dtype=np.int32), np.array(list(rules.bias), dtype=np.int32), np.array(list(rules.bias.values()), dtype=np.float32),
                 np.zeros(0, dtype=np.uint32) if mask is None else mask]
        at = np.concatenate([[0], np.cumsum([(w.nbytes + 15) // 16 * 16 for w in words])])
        operands = np.zeros(at[-1], dtype=np.uint8)
        for w, lo in zip(words, at):
            operands[lo:lo + w.nbytes] = w.view(np.uint8)
        if operands.size > self._rules_bytes:
            ws.alloc(2, operands.size)
            self._rules_bytes = operands.size
        ws.write(kc.rb(2, 0, operands.size), operands)
        part = [kc.rb(2, int(lo), w.nbytes) if w.nbytes else kc.NONE for w, lo in zip(words, at)]
        bias = part[2:5] if n else [kc.NONE] * 3
        call = kc.LogitRulesCall(kc.rb(0), kc.rb(1), part[0], part[1], *bias, part[5], kc.NONE, kc.rb(0), 1, vocab, vocab, vocab, self._tokens.size, n,
                                 0 if mask is None else 1, 0 if mask is None else mask.size, kc.DTYPE_F32)
        self.backend.dispatch(kc.KernelCall.LogitRules(call), ws)

    def _run_rows(self, tokens, base, want, rule=None):
        """One portion of at most max_rows tokens; logits of the wanted rows, one of them where there is a `rule`."""
        m = self.model
        rows = bucket(len(tokens))
        entry = self._session(self._steps, rows, lambda: m.build_step(rows, self.cache.capacity, self.max_rows, False, weightless=True))
        step_in = np.zeros(4 + rows, dtype=np.int32)
        step_in[0], step_in[1] = base, len(tokens)
        step_in[4:4 + len(tokens)] = tokens
        entry[0].write("step_in", step_in)
        session = self._execute(entry)
        vocab = m.config.vocab
        if rule and len(want) and rows == 1:
            self._apply(session, *rule)
        if rows == 1:
            return session.read("logits", np.float32).reshape(1, vocab)[:len(want)]
        out = np.empty((len(want), vocab), dtype=np.float32)
        for lo in range(0, len(want), self.LOGIT_ROWS):
            part = want[lo:lo + self.LOGIT_ROWS]
            n = bucket(len(part))
            head = self._session(self._heads, n, lambda: m.build_head(n, self.max_rows, weightless=True))
            index = np.zeros(n, dtype=np.int32)
            index[:len(part)] = part
            head[0].write("want", index)
            session = self._execute(head)
            if rule:
                self._apply(session, *rule)
            out[lo:lo + len(part)] = session.read("logits", np.float32).reshape(n, vocab)[:len(part)]
        if not len(want):
            self.backend.synchronize()
        return out

    def step(self, seq, tokens, want=None, rules=None, generated=()):
        """Append `tokens` to sequence `seq` (it takes the cache if nobody holds it) and return f32 logits [wanted, vocab];
        `want` lists places among the tokens, the last one by default. `rules` (TokenRules) are applied to the logits of the step's
        last token, then the only one wanted; `generated` are the tokens at the sequence's end that are not its prompt."""
        tokens = np.asarray(tokens, dtype=np.int32)
        if tokens.ndim != 1 or tokens.size == 0:
            raise ValueError("a step brings at least one token")
        if tokens.min() < 0 or tokens.max() >= self.model.config.vocab:
            raise ValueError("token id outside the vocabulary")
        want = [tokens.size - 1] if want is None else [int(i) for i in want]
        if any(not 0 <= i < tokens.size for i in want):
            raise ValueError("a wanted place lies outside the step's tokens")
        if rules is not None and want != [tokens.size - 1]:
            raise ValueError("rules are for the logits of a step's last token")
        rule = None
        if rules is not None:
            if any(t >= self.model.config.vocab for t in rules.bias):
                raise ValueError("a bias for a token outside the vocabulary")
            if len(generated) > tokens.size + (self.cache.length if self.cache.owner == seq else 0):
                raise ValueError("more generated tokens than the sequence has")
            rule = rules, rules.mask(self.model.config.vocab, generated), generated
        self.cache.acquire(seq)
        self.cache.check(tokens.size)
        if rule:
            rule += (self.cache.length + tokens.size,)
        out = np.empty((len(want), self.model.config.vocab), dtype=np.float32)
        for lo in range(0, tokens.size, self.max_rows):
            part = tokens[lo:lo + self.max_rows]
            mine = [k for k, i in enumerate(want) if lo <= i < lo + part.size]
            self._tokens[self.cache.length:self.cache.length + part.size] = part
            self._sent = min(self._sent, self.cache.length)
            out[mine] = self._run_rows(part, self.cache.length, [want[k] - lo for k in mine], rule)
            self.cache.length += part.size
        return out

    def end(self, seq):
        """Give back what the sequence holds."""
        self.cache.release(seq)


class Sampler:
    """Greedy at temperature 0, otherwise a seeded draw from the `top_k` (0 = all) most likely tokens."""

    def __init__(self, temperature=0.0, top_k=0, seed=0):
        self.temperature, self.top_k = temperature, top_k
        self.rng = np.random.default_rng(seed)

    def __call__(self, logits):
        if self.temperature <= 0.0:
            return int(np.argmax(logits))
        z = logits.astype(np.float64) / self.temperature
        if 0 < self.top_k < z.size:
            z[z < np.partition(z, -self.top_k)[-self.top_k]] = -np.inf
        p = np.exp(z - z.max())
        return int(self.rng.choice(z.size, p=p / p.sum()))


class Request:
    def __init__(self, prompt, max_new_tokens, sampler=None, stop=(), rules=None):
        self.rules = rules         # TokenRules, or None
        self.prompt, self.max_new_tokens, self.sampler, self.stop = list(prompt), max_new_tokens, sampler or Sampler(), frozenset(stop)
        self.tokens = []           # generated so far


class Scheduler:
    """Runs requests one after another over one StepRunner: the prompt in portions, then one token per step."""

    def __init__(self, runner, portion=None):
        self.runner, self.portion = runner, portion or runner.max_rows
        self.queue, self._next = deque(), 0

    def submit(self, request):
        if not request.prompt:
            raise ValueError("an empty prompt")
        if len(request.prompt) + request.max_new_tokens > self.runner.cache.capacity:
            raise CacheFull("the request does not fit the cache")
        self.queue.append((self._next, request))
        self._next += 1
        return self._next - 1

    def run(self):
        """Work the queue off; yields (request number, token) as tokens come."""
        while self.queue:
            seq, r = self.queue.popleft()
            ruled = lambda: {} if r.rules is None else {"rules": r.rules, "generated": r.tokens}
            try:
                for lo in range(0, len(r.prompt), self.portion):
                    part = r.prompt[lo:lo + self.portion]
                    last = lo + len(part) == len(r.prompt)
                    logits = self.runner.step(seq, part, None, **ruled()) if last else self.runner.step(seq, part, [])
                while len(r.tokens) < r.max_new_tokens:
                    token = r.sampler(logits[0])
                    r.tokens.append(token)
                    yield seq, token
                    if token in r.stop or len(r.tokens) == r.max_new_tokens:
                        break
                    logits = self.runner.step(seq, [token], **ruled())
            finally:
                self.runner.end(seq)


def generate(runner, prompt, max_new_tokens, sampler=None, stop=(), portion=None, rules=None):
    """The continuation of one prompt."""
    scheduler = Scheduler(runner, portion)
    request = Request(prompt, max_new_tokens, sampler, stop, rules)
    scheduler.submit(request)
    for _ in scheduler.run():
        pass
    return request.tokens
