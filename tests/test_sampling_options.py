"""Sampling options on the host: what they ask for, what they refuse, and the token array of a request."""
import numpy as np
import pytest

from pulse_infer_b200.engine.request import InferenceRequest
from pulse_infer_b200.sampling import SamplingParams


def test_what_the_options_look_at():
    assert not SamplingParams().edits_logits and not SamplingParams().needs_history
    for kw in (dict(repetition_penalty=1.1), dict(frequency_penalty=-0.5), dict(presence_penalty=1.0)):
        p = SamplingParams(**kw)
        assert p.edits_logits and p.needs_history
    assert SamplingParams(frequency_penalty=0.1).needs_prompt_len and not SamplingParams(presence_penalty=0.1).needs_prompt_len
    for kw in (dict(logit_bias=((3, 1.0),)), dict(banned_tokens=(4,))):
        p = SamplingParams(**kw)
        assert p.edits_logits and not p.needs_history
    assert not SamplingParams(presence_penalty=-1.0).needs_history


@pytest.mark.parametrize("kw", [dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0), dict(repetition_penalty=float("nan")),
                                dict(repetition_penalty=float("inf")), dict(frequency_penalty=float("nan")), dict(grammar=object())])
def test_options_that_are_refused(kw):
    with pytest.raises(ValueError):
        SamplingParams(**kw)


def test_token_array_follows_the_request():
    req = InferenceRequest(0, [5, 6, 7], 500)
    assert req.token_array().tolist() == [5, 6, 7]
    for t in range(100):
        req.add_sampled_token(t, ())
        assert req.token_array().tolist() == req.all_tokens()
    req.add_pending_token()
    assert req.token_array().tolist() == req.all_tokens()
    req.add_pending_token()
    req.token_array()
    req.resolve_pending_token(77, ())
    assert req.token_array().tolist() == req.all_tokens() and req.token_array()[-2] == 77
    req.drop_pending_tokens()
    assert req.token_array().tolist() == req.all_tokens()
    req.preempt()
    req.add_sampled_token(9, ())
    assert req.token_array().tolist() == req.all_tokens() and req.token_array().dtype == np.int32


@pytest.mark.parametrize("kw", [dict(logit_bias=((3, float("nan")),)), dict(logit_bias=((3, float("inf")),)), dict(logit_bias=((3, 1e39),)),
                                dict(logit_bias=((3, -1e39),)), dict(logit_bias=(3,)), dict(logit_bias=(("a", 1.0),)), dict(logit_bias=((3, None),)),
                                dict(banned_tokens=("a",)), dict(banned_tokens=(None,)), dict(logit_bias=((3, 1.0, 2.0),)), dict(logit_bias=7),
                                dict(repetition_penalty=1e39), dict(repetition_penalty=1e-50), dict(repetition_penalty=1e-39),
                                dict(frequency_penalty=1e39), dict(frequency_penalty=-1e39)])
def test_rules_that_32_bits_cannot_hold_or_that_are_no_rules_are_refused(kw):
    """When the options are made, not in the middle of a step that other requests share."""
    with pytest.raises(ValueError):
        SamplingParams(**kw)


def test_rules_that_are_taken():
    p = SamplingParams(logit_bias={7: 1, np.int64(8): -float("inf")}, banned_tokens=[np.int32(4), 2 ** 40, -1])
    assert p.logit_bias == ((7, 1.0), (8, -float("inf"))) and p.banned_tokens == (4, 2 ** 40, -1)
    assert SamplingParams(logit_bias=[[5, 2.0], (6, 3e38)]).logit_bias == ((5, 2.0), (6, 3e38))
    assert SamplingParams(presence_penalty=float("inf")).needs_history


def test_a_grammar_may_fill_the_same_array_every_time():
    class Shared:
        words = np.zeros(3, dtype=np.int32)

        def token_mask(self, generated):
            self.words[:] = len(generated)
            return self.words

    p = SamplingParams(grammar=Shared())
    masks = [p.token_mask([0] * n, 96) for n in (1, 2, 3)]
    assert [m.tolist() for m in masks] == [[n] * 3 for n in (1, 2, 3)]
