"""Choosing a token where rules have forbidden all or most of them, or forced one."""
import numpy as np
import pytest
import torch

from gpu_util import need_gpu

pytestmark = pytest.mark.gpu
INF = float("inf")
VOCABS = [1, 31, 515, 4097, 20000, 151936]          # one block a row, and rows cut into slices


def _ops():
    from pulse_infer_b200 import ops
    return ops


def _sample(ops, dev, logits, temp, k, p, seed=1, counters=None):
    n = logits.shape[0]
    full = lambda v, dt: torch.full((n,), v, dtype=dt, device=dev)  # noqa: E731
    counters = list(range(n)) if counters is None else counters
    return ops.sample(logits.to(dev), full(temp, torch.float32), full(k, torch.int32), full(p, torch.float32), full(seed, torch.int64),
                      torch.tensor(counters, dtype=torch.int64, device=dev)).cpu().tolist()


@pytest.mark.parametrize("vocab", VOCABS)
def test_a_row_with_nothing_left_gives_no_token(vocab):
    """All -inf, or -inf and NaN: -1, whatever the options; the rows beside it are what they are alone."""
    dev, ops = need_gpu(), _ops()
    g = torch.Generator().manual_seed(vocab)
    rows = torch.randn(5, vocab, generator=g)
    rows[1] = -INF
    rows[3] = torch.where(torch.rand(vocab, generator=g) < 0.5, -INF, float("nan"))
    assert ops.argmax(rows.to(dev)).cpu().tolist()[1::2] == [-1, -1]
    assert ops.argmax(rows.to(dev)).cpu().tolist()[::2] == ops.argmax(rows[::2].contiguous().to(dev)).cpu().tolist()
    for temp, k, p in ((0.0, 0, 0.0), (0.8, 0, 0.0), (1.0, 5, 0.0), (1.0, 0, 0.9), (0.5, 3, 0.5)):
        got = _sample(ops, dev, rows, temp, k, p)
        assert got[1::2] == [-1, -1], (temp, k, p)
        assert got[::2] == _sample(ops, dev, rows[::2].contiguous(), temp, k, p, counters=[0, 2, 4])


@pytest.mark.parametrize("vocab", VOCABS)
def test_an_infinite_logit_is_chosen(vocab):
    """A logit of +inf has all of the probability; of several the first one."""
    dev, ops = need_gpu(), _ops()
    rows = torch.randn(2, vocab, generator=torch.Generator().manual_seed(vocab))
    rows[:, vocab // 2] = INF
    rows[1, vocab - 1] = INF
    rows[1, 0] = float("nan") if vocab > 2 else INF
    want = [vocab // 2] * 2
    assert ops.argmax(rows.to(dev)).cpu().tolist() == want
    for temp, k, p in ((0.8, 0, 0.0), (1.0, 5, 0.0), (1.0, 0, 0.9), (0.5, 3, 0.5)):
        assert _sample(ops, dev, rows, temp, k, p) == want, (temp, k, p)


def test_a_sampler_without_a_choice_gives_minus_one(vocab=2077):
    """Through the sampler: masks and biases that leave nothing, greedy and with a temperature, beside rows that are free."""
    from pulse_infer_b200.sampling import Sampler, SamplingParams
    dev = need_gpu()

    class Nothing:
        def token_mask(self, generated):
            return np.zeros((vocab + 31) // 32, dtype=np.uint32)

    x = torch.randn(5, vocab, generator=torch.Generator().manual_seed(0))
    every = tuple(range(vocab))
    params = [SamplingParams(grammar=Nothing()), SamplingParams(), SamplingParams(grammar=Nothing(), temperature=0.7, top_k=9),
              SamplingParams(banned_tokens=every, temperature=1.0), SamplingParams(banned_tokens=every[1:], temperature=1.0, top_p=0.9)]
    got = Sampler(dev).sample(x.to(dev), params, [0] * 5, [[]] * 5, [0] * 5)
    assert got == [-1, int(x[1].argmax()), -1, -1, 0]
    greedy = [params[0], params[1], SamplingParams(banned_tokens=every)]
    assert Sampler(dev).sample(x[:3].to(dev), greedy, [0] * 3, [[]] * 3, [0] * 3) == [-1, int(x[1].argmax()), -1]


def test_a_request_without_a_choice_ends_and_the_others_go_on(model_folders):
    from pulse_infer_b200 import Engine
    from tiny_configs import CONFIGS
    need_gpu()
    V = CONFIGS["A"].vocab_size

    class ThreeThenNothing:
        def token_mask(self, generated):
            return np.full((V + 31) // 32, 0xffffffff if len(generated) < 3 else 0, dtype=np.uint32)

    for lookahead in (False, True):
        engine = Engine(model_folders["A"], dtype="float32", page_size=8, num_pages=40, max_batch_size=4, lookahead=lookahead)
        alone = engine.generate([[4, 5]], 8, ignore_eos=True)[0]
        a = engine.add_request([1, 2, 3], 8, ignore_eos=True, grammar=ThreeThenNothing())
        b = engine.add_request([1, 2, 3], 8, ignore_eos=True, grammar=ThreeThenNothing(), temperature=1.0, seed=5)
        c = engine.add_request([4, 5], 8, ignore_eos=True)
        engine.run_until_complete()
        for rid in (a, b):
            assert engine.get_request(rid).finish_reason == "invalid_token"
            out = engine.get_result(rid)
            assert len(out) == 4 and out[3] == -1 and min(out[:3]) >= 0
        assert engine.get_result(c) == alone and engine.get_request(c).finish_reason == "length"
        assert list(engine.get_stats().free_pages) == [40]


@pytest.mark.parametrize("vocab", [31, 515, 40000])
@pytest.mark.parametrize("temp,k,p", [(1.0, 0, 0.0), (0.7, 12, 0.0), (1.0, 0, 0.99), (1.3, 20, 0.9)])
def test_a_forbidden_token_is_never_drawn(vocab, temp, k, p):
    """The draw of (seed 0, counter 345377) is exactly zero, which the first kept token's cumulative weight reaches even if
    it is zero: tokens of logit -inf must not be kept.  Others: whatever the draw and however few are allowed."""
    import plain_model
    dev, ops = need_gpu(), _ops()
    assert plain_model.uniform_from(0, 345377) == 0.0
    g = torch.Generator().manual_seed(vocab)
    row = torch.randn(vocab, generator=g)
    allowed = torch.randperm(vocab - 8, generator=g)[:7] + 4                     # fewer than top-k asks for; not the first, nor the last
    masked = torch.full((vocab,), -INF)
    masked[allowed] = row[allowed]
    counters = [345377] + list(range(200))
    got = _sample(ops, dev, masked.repeat(len(counters), 1), temp, k, p, seed=0, counters=counters)
    assert set(got) <= set(allowed.tolist())
    assert p or k or got[0] == int(allowed.min())
