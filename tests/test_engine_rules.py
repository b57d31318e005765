"""Penalties, biases and grammars in the batched engine (CPU, fake models)."""
import numpy as np
import pytest

from test_engine import FakeModel, V

from woolly_b200.engine import (BatchEngine, GenerationConfig, allowed_mask, apply_rules, pack_rules,
                                sample_next_token)


def run(model, prompts, cfgs, **kw):
    eng = BatchEngine(model, session_factory=model.new_session, **kw)
    ids = [eng.submit(p, c) for p, c in zip(prompts, cfgs)]
    eng.run()
    return [eng.finished[i] for i in ids]


def test_apply_rules_row():
    x = np.array([2.0, -2.0, 1.0, 0.5, -1.0, 3.0], np.float32)
    cfg = GenerationConfig(repetition_penalty=2.0, presence_penalty=0.25, frequency_penalty=0.5,
                           logit_bias={3: 1.5, 0: -0.5})
    got = apply_rules(x, cfg, [0, 1], [2, 2, 4], np.array([1, 1, 1, 1, 1, 0], bool))
    # prompt 0, 1: repetition only; 2 twice, 4 once produced
    want = [1.0 - 0.5, -4.0, 0.5 - 1.0 - 0.25, 2.0, -2.0 - 0.75, -np.inf]
    assert np.array_equal(got, np.float32(want))
    assert x[5] == 3.0  # the model's row is left alone


def test_rules_change_what_is_generated():
    m = FakeModel()
    plain, = run(m, [[5, 6]], [GenerationConfig(max_tokens=6, eos_below=0)])
    ban, = run(m, [[5, 6]], [GenerationConfig(max_tokens=6, eos_below=0,
                                              logit_bias={plain.tokens[0]: -1e9})])
    assert plain.tokens[0] not in ban.tokens
    only, = run(m, [[5, 6]], [GenerationConfig(max_tokens=6, eos_below=0, allowed=lambda t: [10, 20, 30])])
    assert set(only.tokens) <= {10, 20, 30} and len(only.tokens) == 6
    bits = np.zeros(V, bool)
    bits[[10, 20, 30]] = True
    same, = run(m, [[5, 6]], [GenerationConfig(max_tokens=6, eos_below=0, allowed=lambda t: bits)])
    assert same.tokens == only.tokens
    never, = run(m, [[5, 6]], [GenerationConfig(max_tokens=20, eos_below=0, frequency_penalty=1e6)])
    assert len(set(never.tokens)) == 20  # nothing twice


def test_a_grammar_that_ends():
    m = FakeModel()
    cfg = GenerationConfig(max_tokens=9, eos_below=0, allowed=lambda t: [7, 8] if len(t) < 3 else [])
    a, b = run(m, [[3, 4], [9]], [cfg, GenerationConfig(max_tokens=5, eos_below=0)])
    assert len(a.tokens) == 3 and a.reason == "constraint" and set(a.tokens) <= {7, 8}
    assert len(b.tokens) == 5 and m.open == 0
    c, = run(m, [[3]], [GenerationConfig(allowed=lambda t: [])])
    assert c.tokens == [] and c.reason == "constraint"


def test_requests_in_a_batch_do_not_mix():
    cfgs = [GenerationConfig(max_tokens=7, eos_below=0, repetition_penalty=1.5, temperature=0.9, seed=1),
            GenerationConfig(max_tokens=7, eos_below=0),
            GenerationConfig(max_tokens=7, eos_below=0, logit_bias={3: 40.0, 4: 40.5}, presence_penalty=2.0)]
    prompts = [[3, 3, 4], [8], [1, 2, 3, 4, 5]]
    together = [r.tokens for r in run(FakeModel(), prompts, cfgs)]
    alone = [run(FakeModel(), [p], [c])[0].tokens for p, c in zip(prompts, cfgs)]
    assert together == alone


class DeviceModel(FakeModel):
    """decode_sample in numpy, undoing pack_rules' arrays as the operator reads them."""

    def decode_sample(self, sessions, ids, temperature, top_k, top_p, u, rules=None):
        rows = np.stack(self.forward_sessions(sessions, [[i] for i in ids]))
        self.rules = rules
        out = []
        for i, row in enumerate(rows):
            row = row.astype(np.float32)
            if rules is not None:
                p, hs = rules["params"], rules["history_start"]
                h = rules["history"][hs[i]:hs[i + 1]].tolist()
                n = int(rules["prompt_lens"][i])
                bias = {}
                if "bias_start" in rules:
                    b = slice(rules["bias_start"][i], rules["bias_start"][i + 1])
                    bias = dict(zip(rules["bias_tokens"][b].tolist(), rules["bias_values"][b].tolist()))
                mask = None
                if p["allowed_row"][i] >= 0:
                    w = rules["allowed"][p["allowed_row"][i]].view(np.uint32)
                    mask = ((w[np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1).astype(bool)
                row = apply_rules(row, GenerationConfig(
                    repetition_penalty=p["repetition"][i], presence_penalty=p["presence"][i],
                    frequency_penalty=p["frequency"][i], logit_bias=bias), h[:n], h[n:], mask)
            out.append(sample_next_token(row, GenerationConfig(temperature=temperature[i], top_k=top_k[i],
                                                              top_p=top_p[i]), Draw(u[i])))
        return out


class Draw:
    def __init__(self, u):
        self.u = u

    def random(self, dtype=None):
        return self.u


def test_device_sampling_gets_the_same_rules():
    cfgs = [GenerationConfig(max_tokens=8, eos_below=0, repetition_penalty=1.3, temperature=0.8, seed=4),
            GenerationConfig(max_tokens=8, eos_below=0, logit_bias={11: 3.0, 12: 2.0}, frequency_penalty=0.7),
            GenerationConfig(max_tokens=8, eos_below=0),
            GenerationConfig(max_tokens=8, eos_below=0, temperature=1.1, seed=9,
                             allowed=lambda t: range(5, 25) if len(t) < 6 else [])]
    prompts = [[3, 3, 4], [8, 1], [1, 2, 3], [7]]
    host = [(r.tokens, r.reason) for r in run(FakeModel(), prompts, cfgs)]
    m = DeviceModel()
    dev = [(r.tokens, r.reason) for r in run(m, prompts, cfgs, device_sampling=True)]
    assert host == dev and m.rules is not None
    m = DeviceModel()
    run(m, [[5]], [GenerationConfig(max_tokens=4, eos_below=0)], device_sampling=True)
    assert m.rules is None  # nothing asked for: nothing sent


def test_pack_rules_without_requests():
    assert pack_rules([], [], V)["history_start"].tolist() == [0]


@pytest.mark.parametrize("kw", [dict(repetition_penalty=0.0), dict(repetition_penalty=float("nan")),
                                dict(presence_penalty=float("inf")), dict(frequency_penalty=float("nan")),
                                dict(logit_bias={V: 1.0}), dict(logit_bias={-1: 1.0}),
                                dict(logit_bias={3: float("nan")})])
def test_submit_refuses(kw):
    m = FakeModel()
    with pytest.raises(ValueError):
        BatchEngine(m, session_factory=m.new_session).submit([1], GenerationConfig(**kw))


def test_allowed_mask_refuses():
    for ids in ([V], [-1], np.zeros(V + 1, bool)):
        with pytest.raises(ValueError):
            allowed_mask(GenerationConfig(allowed=lambda t: ids), [], V)
