"""Penalties, biases and masks on logits against float64."""
import numpy as np
import pytest
import torch

from gpu_util import need_gpu

pytestmark = pytest.mark.gpu


def _ops():
    from pulse_infer_b200 import ops
    return ops


def plain_rules(x, histories, prompts, rep, freq, pres, biases, masks):
    """x [n, V] float64; per row: history, length of its prompt, penalties, [(token, value)], bool mask [V] or None.
    Returns (result, bound on the error of 32-bit arithmetic): six roundings of numbers not above ``size``."""
    x, size = x.copy(), np.abs(x)
    for r in range(x.shape[0]):
        for v in set(histories[r]):
            if 0 <= v < x.shape[1]:
                count = sum(1 for i, h in enumerate(histories[r]) if h == v and i >= prompts[r])
                x[r, v] = x[r, v] / rep[r] if x[r, v] > 0 else x[r, v] * rep[r]
                size[r, v] = max(size[r, v], abs(x[r, v])) + abs(freq[r] * count) + abs(pres[r])
                x[r, v] -= freq[r] * count + pres[r]
        last = {}
        for v, b in biases[r]:
            last[v] = b
        for v, b in last.items():
            if 0 <= v < x.shape[1]:
                x[r, v] += b
                size[r, v] += abs(b)
        if masks[r] is not None:
            x[r, ~masks[r]] = -np.inf
    return x, 6 * 2.0 ** -24 * size


def _case(rows, V, seed, history=200, with_bias=True, with_mask=True):
    rng = np.random.RandomState(seed)
    x = (3 * rng.randn(rows, V)).astype(np.float32)
    lens = [0 if r == 1 else int(rng.randint(0, history + 1)) for r in range(rows)]
    histories = [[int(v) for v in np.minimum(V * rng.rand(n) ** 3, V - 1)] for n in lens]
    if rows > 2:
        histories[2] += [0, V - 1, V - 1, -1, V, V + 7, 2 ** 31 - 1, -2 ** 31]          # the last ids, and some that are none
    prompts = [int(rng.randint(0, len(h) + 1)) for h in histories]
    f = lambda choices: rng.choice(choices, rows).astype(np.float32)  # noqa: E731
    rep, freq, pres = f([1.0, 1.3, 0.8]), f([0.0, 0.7, -0.2]), f([0.0, 1.5])
    biases = [[] for _ in range(rows)]
    if with_bias:
        biases = [[(int(v), float(np.float32(rng.randn()))) for v in rng.randint(0, V, rng.randint(0, 40))] for _ in range(rows)]
        biases[0] += [(0, 1.0), (V - 1, -2.0), (0, 3.0), (-5, 1.0), (V, 1.0), (V - 1, -float("inf"))]
    masks = [None if not with_mask or r % 3 == 0 else rng.rand(V) < 0.5 for r in range(rows)]
    if with_mask and rows > 4:
        masks[4] = np.zeros(V, dtype=bool)                                               # nothing is left
    return x, histories, prompts, rep, freq, pres, biases, masks


def _tensors(dev, V, histories, prompts, rep, freq, pres, biases, masks):
    i32 = lambda v: torch.tensor(np.asarray(v, dtype=np.int64).astype(np.int32), device=dev)  # noqa: E731
    f32 = lambda v: torch.tensor(np.asarray(v, dtype=np.float32), device=dev)  # noqa: E731
    off = lambda rows: i32(np.concatenate([[0], np.cumsum([len(r) for r in rows])]))  # noqa: E731
    flat = lambda rows: [v for r in rows for v in r]  # noqa: E731
    args = [i32(flat(histories)), off(histories), i32(prompts), f32(rep), f32(freq), f32(pres)]
    kw = {}
    if any(biases):
        kw.update(bias_off=off(biases), bias_tokens=i32([v for v, _ in flat(biases)]), bias_values=f32([b for _, b in flat(biases)]))
    held = [m for m in masks if m is not None]
    if held:
        words = np.zeros((len(held), (V + 31) // 32 * 32), dtype=bool)
        words[:, V:] = True
        for i, m in enumerate(held):
            words[i, :V] = m
        words = np.packbits(words, axis=1, bitorder="little").view(np.uint32).view(np.int32)
        at, rows = 0, []
        for m in masks:
            rows.append(-1 if m is None else at)
            at += m is not None
        kw.update(mask=torch.tensor(words.copy(), device=dev), mask_row=i32(rows))
    return args, kw


@pytest.mark.parametrize("rows,V", [(1, 151936), (5, 4096), (7, 4097), (3, 1), (6, 31), (9, 515), (5, 12291), (130, 2077), (4, 6144), (4, 6145)])
@pytest.mark.parametrize("with_bias,with_mask", [(True, True), (False, False), (True, False), (False, True)])
def test_logit_rules(rows, V, with_bias, with_mask):
    dev, ops = need_gpu(), _ops()
    x, *rules = _case(rows, V, rows + V, with_bias=with_bias, with_mask=with_mask)
    want, bound = plain_rules(x.astype(np.float64), *rules)
    args, kw = _tensors(dev, V, *rules)
    src = torch.tensor(x, device=dev)
    out = ops.logit_rules(src, *args, **kw)
    assert torch.equal(src.cpu(), torch.tensor(x))
    got = out.cpu().double().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)) and np.array_equal(got[~fine], want[~fine])
    assert (np.abs(got[fine] - want[fine]) <= bound[fine]).all()
    # in place, and between rows that are further apart than the vocabulary
    assert torch.equal(ops.logit_rules(src, *args, **kw, out=src), out) and torch.equal(src, out)
    wide = torch.full((rows, V + 3), 5.0, device=dev)
    wide[:, :V] = torch.tensor(x, device=dev)
    apart = torch.full((rows, V + 7), 6.0, device=dev)
    ops.logit_rules(wide[:, :V], *args, **kw, out=apart[:, :V])
    assert torch.equal(apart[:, :V], out) and (apart[:, V:] == 6).all() and (wide[:, V:] == 5).all()


def test_logit_rules_long_history_and_special_logits():
    dev, ops = need_gpu(), _ops()
    V, L = 5000, 70000
    x, *rules = _case(2, V, 3, with_bias=False, with_mask=False)
    rng = np.random.RandomState(0)
    rules[0] = [[int(v) for v in rng.randint(0, 50, L)], [7] * 3]
    rules[1] = [1000, 1]
    x[0, 3], x[0, 4], x[1, 7] = -np.inf, np.inf, 0.0
    want, bound = plain_rules(x.astype(np.float64), *rules)
    args, kw = _tensors(dev, V, *rules)
    got = ops.logit_rules(torch.tensor(x, device=dev), *args, **kw).cpu().double().numpy()
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine]) and (np.abs(got[fine] - want[fine]) <= bound[fine]).all()


def test_logit_rules_in_a_graph():
    dev, ops = need_gpu(), _ops()
    x, *rules = _case(4, 9000, 8)
    args, kw = _tensors(dev, 9000, *rules)
    src = torch.tensor(x, device=dev)
    want = ops.logit_rules(src, *args, **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.logit_rules(src, *args, **kw)
    got.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_what_logit_rules_refuses():
    from pulse_infer_b200.ops import KernelError
    dev, ops = need_gpu(), _ops()
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)  # noqa: E731
    f32 = lambda *shape: torch.zeros(shape, device=dev)  # noqa: E731
    base = dict(logits=f32(2, 70), history=i32(0), history_off=i32(3), prompt_len=i32(2), repetition=f32(2) + 1, frequency=f32(2), presence=f32(2))
    ops.logit_rules(**base)
    assert ops.logit_rules(**{**base, "logits": f32(0, 70), "history_off": i32(1), "prompt_len": i32(0), "repetition": f32(0), "frequency": f32(0),
                              "presence": f32(0)}).shape == (0, 70)
    for kw in (dict(logits=f32(2, 70).bfloat16()), dict(logits=f32(70, 2).T), dict(logits=f32(70)), dict(history=i32(1).long()), dict(history_off=i32(2)),
               dict(prompt_len=i32(3)), dict(repetition=i32(2)), dict(frequency=f32(4)[::2]), dict(presence=f32(1)), dict(bias_off=i32(3)),
               dict(bias_off=i32(3), bias_tokens=i32(2), bias_values=f32(1)), dict(bias_off=i32(2), bias_tokens=i32(1), bias_values=f32(1)),
               dict(mask=i32(1, 3)), dict(mask=i32(1, 2), mask_row=i32(2)), dict(mask=i32(1, 3), mask_row=i32(1)), dict(mask=i32(3), mask_row=i32(2)),
               dict(out=f32(2, 71)), dict(out=f32(2, 70).double()), dict(presence=torch.zeros(2))):
        with pytest.raises(KernelError):
            ops.logit_rules(**{**base, **kw})


class _Grammar:
    """Allows, after k generated tokens, the ids that are k modulo 7; everything after the fourth."""

    def __init__(self, vocab):
        self.vocab, self.seen = vocab, []

    def token_mask(self, generated):
        self.seen.append(list(generated))
        if len(generated) >= 4:
            return None
        bits = np.zeros((self.vocab + 31) // 32 * 32, dtype=bool)
        bits[len(generated):self.vocab:7] = True
        return np.packbits(bits, bitorder="little").view(np.uint32)


def test_sampler_applies_the_rules_of_every_request():
    from pulse_infer_b200.sampling import Sampler, SamplingParams
    dev = need_gpu()
    V = 2077
    x = (3 * np.random.RandomState(4).randn(7, V)).astype(np.float32)
    grammar = _Grammar(V)
    params = [SamplingParams(), SamplingParams(presence_penalty=1.5), SamplingParams(repetition_penalty=1.3, frequency_penalty=0.7),
              SamplingParams(banned_tokens=(3, 5, 3), logit_bias=((9, 4.0), (3, 2.0))), SamplingParams(grammar=grammar),
              SamplingParams(presence_penalty=0.3, repetition_penalty=0.9, frequency_penalty=0.2, logit_bias=((1, -1.0),), banned_tokens=(0,)),
              SamplingParams(temperature=0.7, top_k=5, presence_penalty=2.0, seed=3)]
    histories = [[], [1, 2, 2, 3], [4, 4, 5, 6, 6], [3, 9], [8, 8, 2], list(range(50)) * 2, [int(np.argmax(x[6]))]]
    prompts = [0, 4, 2, 0, 1, 50, 0]
    rep = [p.repetition_penalty for p in params]
    freq = [p.frequency_penalty for p in params]
    pres = [p.presence_penalty for p in params]
    biases = [list(p.logit_bias) + [(t, -np.inf) for t in p.banned_tokens] for p in params]
    masks = [None] * 7
    masks[4] = np.arange(V) % 7 == 2
    used = [h if p.needs_history else [] for h, p in zip(histories, params)]
    want, _ = plain_rules(x.astype(np.float64), used, prompts, rep, freq, pres, biases, masks)
    src = torch.tensor(x, device=dev)
    sampler = Sampler(dev)
    got = sampler.sample(src, params, [0] * 7, histories, prompts)
    assert got[:6] == [int(np.argmax(w)) for w in want[:6]] and torch.equal(src.cpu(), torch.tensor(x))
    assert got[6] in np.argsort(-want[6])[:5] and grammar.seen == [[8, 2]]
    # as before: no history, no penalty; presence alone without the lengths of the prompts
    assert sampler.sample(src[1:2], [params[1]], [0]) == [int(np.argmax(x[1]))]
    assert sampler.sample(src[1:2], [params[1]], [0], [histories[1]]) == [int(np.argmax(want[1]))]
    bad = _Grammar(V)
    bad.token_mask = lambda generated: np.zeros(3, dtype=np.int32)
    with pytest.raises(ValueError, match="token mask"):
        sampler.sample(src[:1], [SamplingParams(grammar=bad)], [0], [[]], [0])


def test_engine_generates_under_rules(model_folders):
    """Through Engine: a grammar sees what was generated, a repeated token is penalised out, biases choose."""
    from pulse_infer_b200 import Engine
    from tiny_configs import CONFIGS
    need_gpu()
    V = CONFIGS["A"].vocab_size
    engine = Engine(model_folders["A"], dtype="float32", page_size=8, num_pages=40, max_batch_size=4)
    grammar = _Grammar(V)
    a = engine.add_request([1, 2, 3], 6, ignore_eos=True, grammar=grammar)
    b = engine.add_request([4, 5], 12, ignore_eos=True, frequency_penalty=1e4)
    c = engine.add_request([4, 5], 5, ignore_eos=True, logit_bias={17: 1e4})
    d = engine.add_request([4, 5], 12, ignore_eos=True, repetition_penalty=1e6)
    engine.run_until_complete()
    out = [engine.get_result(i) for i in (a, b, c, d)]
    assert [t % 7 for t in out[0][:4]] == [0, 1, 2, 3] and grammar.seen == [out[0][:i] for i in range(6)]
    assert len(set(out[1])) == 12 and out[2] == [17] * 5
    assert len(out[3]) == 12


def test_logit_rules_rows_that_overlap_are_refused_and_one_row_may_have_any_stride():
    from pulse_infer_b200.ops import KernelError
    dev, ops = need_gpu(), _ops()
    V = 100
    x, *rules = _case(2, V, 4, with_bias=False, with_mask=False)
    args, _ = _tensors(dev, V, *rules)
    with pytest.raises(KernelError):
        ops.logit_rules(torch.zeros(1, V, device=dev).expand(2, V), *args)
    with pytest.raises(KernelError):
        ops.logit_rules(torch.zeros(2, V, device=dev), *args, out=torch.zeros(1, V, device=dev).expand(2, V))
    one = [[r[0]] if isinstance(r, list) else r[:1] for r in rules]
    args, _ = _tensors(dev, V, *one)
    src = torch.tensor(x[:1], device=dev)
    odd = torch.empty_strided((1, V), (3, 1), device=dev)
    odd.copy_(src)
    assert torch.equal(ops.logit_rules(odd, *args), ops.logit_rules(src, *args))


def test_a_bias_of_minus_infinity_forbids_whatever_the_logit_is():
    dev, ops = need_gpu(), _ops()
    x = torch.zeros(2, 40, device=dev)
    x[0, 5], x[0, 6], x[0, 7], x[1, 5] = float("inf"), float("nan"), 2.0, float("inf")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    one, none = torch.ones(2, device=dev), torch.zeros(2, device=dev)
    out = ops.logit_rules(x, i32([]), i32([0, 0, 0]), i32([0, 0]), one, none, none, bias_off=i32([0, 3, 3]), bias_tokens=i32([5, 6, 7]),
                          bias_values=torch.full((3,), -float("inf"), device=dev))
    assert (out[0, 5:8] == -float("inf")).all() and (out[0, :5] == 0).all() and (out[0, 8:] == 0).all() and out[1, 5] == float("inf")


def test_logit_rules_output_that_overlaps_the_logits():
    from pulse_infer_b200.ops import KernelError
    dev, ops = need_gpu(), _ops()
    i32 = lambda n: torch.zeros(n, dtype=torch.int32, device=dev)  # noqa: E731
    rules = (i32(0), i32(4), i32(3), torch.ones(3, device=dev), torch.zeros(3, device=dev), torch.zeros(3, device=dev))
    flat = torch.randn(1000, device=dev)
    view = lambda at, ld: flat.as_strided((3, 70), (ld, 1), at)  # noqa: E731
    for a, b in (((0, 80), (1, 80)), ((4, 80), (0, 80)), ((0, 80), (0, 90)), ((0, 80), (200, 80)), ((100, 200), (31, 200)), ((0, 70), (139, 70))):
        with pytest.raises(KernelError):
            ops.logit_rules(view(*a), *rules, out=view(*b))
    for a, b in (((0, 80), (0, 80)), ((0, 200), (70, 200)), ((100, 200), (30, 200)), ((0, 70), (210, 70)), ((300, 80), (60, 80))):
        want = view(*a).clone()
        assert torch.equal(ops.logit_rules(view(*a), *rules, out=view(*b)), want)


def test_ids_that_no_vocabulary_has_are_passed_over():
    """Through the sampler, also where 32 bits do not hold them."""
    from pulse_infer_b200.sampling import Sampler, SamplingParams
    dev = need_gpu()
    V = 300
    x = torch.randn(2, V, generator=torch.Generator().manual_seed(1))
    best = int(x[0].argmax())
    odd = (2 ** 40, -1, -2 ** 40, V, 2 ** 31, -2 ** 31 - 1, 2 ** 32 + best)
    got = Sampler(dev).sample(x.to(dev), [SamplingParams(banned_tokens=odd, logit_bias=tuple((t, 50.0) for t in odd)),
                                          SamplingParams(banned_tokens=odd + (int(x[1].argmax()),))], [0, 0])
    assert got == [best, int(x[1].topk(2).indices[1])]


@pytest.mark.parametrize("lookahead", [False, True])
def test_a_grammar_that_fails_ends_its_own_request_only(model_folders, lookahead):
    """One that raises, one whose mask has another size, one whose mask is of another type: each ends its request with what it
    generated so far; the others, and a later request, get what they get alone."""
    import warnings
    from pulse_infer_b200 import Engine
    from tiny_configs import CONFIGS
    need_gpu()
    V = CONFIGS["A"].vocab_size

    class Fails(_Grammar):
        def __init__(self, how, after):
            super().__init__(V)
            self.how, self.after = how, after

        def token_mask(self, generated):
            mask = super().token_mask(generated)
            return mask if len(generated) < self.after else self.how()

    def raises():
        raise RuntimeError("no such state")

    engine = Engine(model_folders["A"], dtype="float32", page_size=8, num_pages=60, max_batch_size=6, lookahead=lookahead)
    alone = engine.generate([[4, 5]], 7, ignore_eos=True)[0]
    ids = [engine.add_request([1, 2, 3], 6, ignore_eos=True, grammar=Fails(how, after))
           for how, after in ((raises, 2), (lambda: np.zeros(3, np.int32), 0), (lambda: np.zeros((V + 31) // 32, np.int64), 1), (lambda: "no", 3))]
    free = engine.add_request([4, 5], 7, ignore_eos=True)
    good = engine.add_request([1, 2, 3], 6, ignore_eos=True, grammar=_Grammar(V))
    with warnings.catch_warnings(record=True) as told:
        warnings.simplefilter("always")
        engine.run_until_complete()
    assert [len(engine.get_result(i)) for i in ids] == [2, 0, 1, 3]
    assert [engine.get_request(i).finish_reason for i in ids] == ["grammar_error"] * 4
    assert sum("grammar" in str(w.message) for w in told) == 4 and any("no such state" in str(w.message) for w in told)
    assert engine.get_result(free) == alone and len(engine.get_result(good)) == 6
    assert [t % 7 for t in engine.get_result(good)[:4]] == [0, 1, 2, 3]
    assert engine.generate([[4, 5]], 7, ignore_eos=True)[0] == alone and list(engine.get_stats().free_pages) == [60]


def test_engine_applies_repetition_penalties_to_prompt_and_output(model_folders):
    """Greedy tokens of an engine against a loop on the host that penalises the logits which the engine saw."""
    from pulse_infer_b200 import Engine
    need_gpu()
    engine = Engine(model_folders["A"], dtype="float32", page_size=8, num_pages=40, max_batch_size=4)
    plain = engine.generate([[4, 5, 6]], 16, ignore_eos=True)[0]
    for kw in (dict(repetition_penalty=1.5), dict(repetition_penalty=1e6), dict(repetition_penalty=0.5), dict(repetition_penalty=1.2, presence_penalty=0.3)):
        seen = []
        engine.engine.logits_hook = lambda reqs, logits: seen.append(logits[0].double().cpu().numpy())
        out = engine.generate([[4, 5, 6]], 16, ignore_eos=True, **kw)[0]
        engine.engine.logits_hook = None
        history = [4, 5, 6]
        for x, token in zip(seen, out):
            for t in set(history):
                x[t] = (x[t] / kw["repetition_penalty"] if x[t] > 0 else x[t] * kw["repetition_penalty"]) - kw.get("presence_penalty", 0.0)
            assert token == int(np.argmax(x))
            history.append(token)
        # a penalty of 1e6 leaves no token that was there; the mild ones need not change what this model repeats
        assert len(seen) == len(out) == 16 and (kw["repetition_penalty"] < 1e6 or (out != plain and len(set(out)) == 16))


def test_a_sampler_takes_rules_for_rows_that_share_their_logits():
    """One row of logits expanded to several requests, as before there was a kernel for all rules."""
    from pulse_infer_b200.sampling import Sampler, SamplingParams
    dev = need_gpu()
    x = torch.randn(1, 900, generator=torch.Generator().manual_seed(2))
    first, second, third = x[0].topk(3).indices.tolist()
    params = [SamplingParams(banned_tokens=(first,)), SamplingParams(), SamplingParams(banned_tokens=(first, second))]
    assert Sampler(dev).sample(x.to(dev).expand(3, 900), params, [0] * 3) == [second, first, third]
