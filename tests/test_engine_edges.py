"""The batched engine where rules close every token, where they reach the ends
of f32, and where a caller's function raises (CPU, fake models)."""
import numpy as np
import pytest

from test_engine import FakeModel, V
from test_engine_rules import DeviceModel, run

from woolly_b200.engine import BatchEngine, GenerationConfig

INF = float("inf")
LOWEST = float(np.finfo(np.float32).min)


def both(prompts, cfgs):
    """Tokens and reasons with host sampling, which the other path must repeat."""
    host = [(r.tokens, r.reason) for r in run(FakeModel(), prompts, cfgs())]
    m = DeviceModel()
    assert [(r.tokens, r.reason) for r in run(m, prompts, cfgs(), device_sampling=True)] == host
    assert m.open == 0
    return host


@pytest.mark.parametrize("temperature", [0.0, 0.7])
@pytest.mark.parametrize("low", [-INF, LOWEST, -1e39])
def test_a_bias_that_closes_all_that_a_grammar_allows(temperature, low):
    """The request ends, at once or on the way; the others go on."""
    def cfgs():
        return [GenerationConfig(max_tokens=5, eos_below=0, temperature=temperature, logit_bias={5: low},
                                 allowed=lambda t: [5]),
                GenerationConfig(max_tokens=5, eos_below=0, temperature=temperature, logit_bias={5: low},
                                 allowed=lambda t: [5] if len(t) > 2 else [4, 5, 6]),
                GenerationConfig(max_tokens=5, eos_below=0)]
    got = both([[3], [4], [9]], cfgs)
    assert got[0] == ([], "constraint")
    assert got[1][1] == "constraint" and len(got[1][0]) == 3 and set(got[1][0]) <= {4, 6}
    assert len(got[2][0]) == 5


@pytest.mark.parametrize("low", [-INF, LOWEST])
def test_a_bias_closes_its_token(low):
    plain = both([[5, 6]], lambda: [GenerationConfig(max_tokens=6, eos_below=0)])[0][0]
    got = both([[5, 6]], lambda: [GenerationConfig(max_tokens=6, eos_below=0, temperature=1.0,
                                                   logit_bias={plain[0]: low, plain[1]: low})])[0][0]
    assert len(got) == 6 and not set(got) & set(plain[:2])
    every = both([[5, 6]], lambda: [GenerationConfig(logit_bias=dict.fromkeys(range(V), low))])[0]
    assert every == ([], "constraint")


@pytest.mark.parametrize("kw", [dict(logit_bias={5: 1e30}), dict(repetition_penalty=1e30),
                                dict(repetition_penalty=1e-30), dict(frequency_penalty=1e30),
                                dict(frequency_penalty=-1e30, presence_penalty=-1e30)])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_the_largest_rules_leave_a_choice(kw, temperature):
    got = both([[5, 7]], lambda: [GenerationConfig(max_tokens=8, eos_below=0, temperature=temperature,
                                                   allowed=lambda t: [5, 7, 9], **kw)])[0][0]
    assert len(got) == 8 and set(got) <= {5, 7, 9}


@pytest.mark.parametrize("kw", [dict(logit_bias={5: INF}), dict(logit_bias={5: 1e31}), dict(logit_bias={5: 1e39}),
                                dict(repetition_penalty=1e31), dict(repetition_penalty=1e-31),
                                dict(presence_penalty=2e30), dict(frequency_penalty=-2e30)])
def test_submit_refuses_what_f32_cannot_hold(kw):
    m = FakeModel()
    with pytest.raises(ValueError):
        BatchEngine(m, session_factory=m.new_session).submit([1], GenerationConfig(**kw))
