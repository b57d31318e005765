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


class Stop(Exception):
    pass


def raises_at(n, ids=range(V)):
    """A grammar that raises once n tokens are there."""
    def allowed(tokens):
        if len(tokens) == n:
            raise Stop
        return ids
    return allowed


def drain(eng):
    """Steps until all is finished; the number of steps that raised."""
    raised = 0
    for _ in range(100):
        if eng.idle():
            return raised
        try:
            eng.step()
        except Stop:
            raised += 1
    raise AssertionError("requests that never finish")


@pytest.mark.parametrize("model,device", [(FakeModel, False), (DeviceModel, True)])
@pytest.mark.parametrize("at", [0, 1, 3])
def test_a_grammar_that_raises_ends_its_own_request(model, device, at):
    """On the first token, where the request has just been admitted, or later:
    the others' tokens are those of a run without it, and all sessions close."""
    cfg = lambda **kw: GenerationConfig(max_tokens=6, eos_below=0, temperature=0.8, **kw)  # noqa: E731
    prompts = [[3, 4], [8], [9, 9], [2, 7]]
    alone = [run(model(), [p], [cfg(seed=i)], device_sampling=device)[0].tokens for i, p in enumerate(prompts)]
    m = model()
    eng = BatchEngine(m, session_factory=m.new_session, device_sampling=device)
    ids = [eng.submit(p, cfg(seed=i, allowed=raises_at(at)) if i == 1 else cfg(seed=i))
           for i, p in enumerate(prompts)]
    assert drain(eng) == 1
    assert m.open == 0
    got = [eng.finished[i] for i in ids]
    assert [r.tokens for i, r in enumerate(got) if i != 1] == [t for i, t in enumerate(alone) if i != 1]
    assert got[1].reason == "error" and got[1].tokens == alone[1][:at]


@pytest.mark.parametrize("model,device", [(FakeModel, False), (DeviceModel, True)])
@pytest.mark.parametrize("at", [1, 2, 5])
def test_a_callback_that_raises_costs_no_token(model, device, at):
    seen = []

    def callback(rid, tok, done, reason):
        seen.append((rid, tok))
        if rid == 0 and sum(r == 0 for r, _ in seen) == at:
            raise Stop
    m = model()
    eng = BatchEngine(m, session_factory=m.new_session, device_sampling=device)
    cfg = GenerationConfig(max_tokens=5, eos_below=0)
    ids = [eng.submit([p], cfg, on_token=callback) for p in (3, 8)]
    assert drain(eng) == 1 and m.open == 0
    for i, p in zip(ids, (3, 8)):
        want = run(model(), [[p]], [cfg])[0].tokens
        assert eng.finished[i].tokens == want == [t for r, t in seen if r == i]
        assert eng.finished[i].reason == "length"


def test_a_prefill_that_raises_leaves_the_other_requests():
    class Broken(FakeModel):
        def forward_sessions(self, sessions, ids):
            if any(13 in i for i in ids):
                raise Stop
            return super().forward_sessions(sessions, ids)
    m = Broken()
    eng = BatchEngine(m, session_factory=m.new_session)
    cfg = GenerationConfig(max_tokens=3, eos_below=0, allowed=lambda t: [1, 2])
    ids = [eng.submit(p, cfg) for p in ([13], [5], [6, 13], [7])]
    assert drain(eng) == 1 and m.open == 0
    assert [eng.finished[i].reason for i in ids] == ["error", "length", "error", "length"]


def test_a_session_that_cannot_be_made_keeps_those_admitted():
    m = FakeModel()

    def factory():
        if m.open == 1 and factory.broken:
            factory.broken = False
            raise Stop
        return m.new_session()
    factory.broken = True
    eng = BatchEngine(m, session_factory=factory)
    cfg = GenerationConfig(max_tokens=3, eos_below=0)
    ids = [eng.submit([p], cfg) for p in (4, 5)]
    assert drain(eng) == 1 and m.open == 0
    assert [len(eng.finished[i].tokens) for i in ids] == [3, 3]
