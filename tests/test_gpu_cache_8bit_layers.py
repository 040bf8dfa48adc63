"""The whole layer path over an 8-bit cache, with the quantisation taken out of the comparison: after a step the engine's own
pages are read back, and the plain implementation attends over those keys and values, in 64 bits.  What is left between the two
is what bfloat16 pages leave, so the tolerance is theirs."""
import dataclasses

import numpy as np
import pytest
import torch

import plain_model
from gpu_util import need_gpu
from helpers import load_plain, random_tokens
from tiny_configs import CONFIGS

pytestmark = pytest.mark.gpu
TOL = 2e-2                 # of the largest |logit|: the tests' tolerance for bfloat16


def _pages(runner, request, cache, tokens):
    """Keys and values [tokens, kv heads, d] of a request in one cache, float64; zeros where a page was given back."""
    from pulse_infer_b200 import ops
    group = runner.cache.group_for_cache(cache)
    page = runner.cache.page_size
    ids = group.device_table[runner.cache.slot(request), :(tokens + page - 1) // page].contiguous()
    keys, values = ops.pages_8bit_to_bf16(*group.kv(cache), *group.scales(cache), ids)
    return tuple(x.double().cpu().transpose(1, 2).flatten(0, 1)[:tokens].numpy() for x in (keys, values))


def _forward_on_pages(runner, request, folder, tokens, order, monkeypatch, edit=None):
    """The plain logits of ``tokens`` with every cache's keys and values as the pages hold them."""
    cfg, w = load_plain(folder)
    order = order or [(i, i) for i in range(cfg["num_hidden_layers"])]
    writers = iter([c for layer, c in order if f"model.layers.{layer}.self_attn.k_proj.weight" in w])

    def stored(*args, **kw):
        k, v = _pages(runner, request, next(writers), len(tokens))
        return (k, v) if edit is None else edit(k, v)
    with monkeypatch.context() as m:
        m.setattr(plain_model, "layer_keys_values", stored)
        return plain_model.forward(cfg, w, tokens, order=order)


def _run_cuts(runner, folder, vocab, order, monkeypatch):
    """A prompt, single tokens, portions beside another request that decodes; every step against the pages it left."""
    from pulse_infer_b200.engine import Segment
    toks = random_tokens(7, 330, vocab)
    runner.open("a"); runner.open("x")
    runner.step([Segment("x", random_tokens(9, 21, vocab), [])])
    at = 0
    for n in (200, 1, 1, 13, 1, 2, 31, 1, 70, 1):
        beside = [] if n == 200 else [Segment("x", [(3 * at) % vocab], [])]
        got = runner.step(beside + [Segment("a", toks[at:at + n], list(range(n)))]).double().cpu().numpy()
        at += n
        want = _forward_on_pages(runner, "a", folder, toks[:at], order, monkeypatch)[at - n:]
        scale = np.abs(want).max()
        assert np.abs(got - want).max() <= TOL * scale, (at, n, np.abs(got - want).max() / scale)
    # the bound means something: values of one block of 16 tokens that are lost move the last logits beyond it
    last = runner.step([Segment("a", [toks[at]], [0])]).double().cpu().numpy()
    at += 1
    moved = []
    for block in range(0, at, 64):
        def lose(k, v):
            v = v.copy()
            v[block:block + 16] = 0
            return k, v
        want = _forward_on_pages(runner, "a", folder, toks[:at], order, monkeypatch, lose)[-1:]
        moved.append(np.abs(last - want).max() / np.abs(want).max())
    assert max(moved) > 2 * TOL, moved
    runner.check_device_errors()


@pytest.mark.parametrize("dtype", ["float8_e4m3fn", "int8"])
@pytest.mark.parametrize("name,page,graphs", [("D", 16, False), ("E", 16, True), ("E", 64, False), ("D", 128, True)])
def test_steps_against_their_own_pages(name, page, graphs, dtype, model_folders, monkeypatch):
    from pulse_infer_b200.engine import build_runner
    need_gpu()
    runner = build_runner(model_folders[name], dtype="bfloat16", device="cuda:0", page_size=page, num_pages=96, max_requests=4,
                          max_tokens_per_request=512, cache_dtype=dtype, use_cuda_graphs=graphs)
    _run_cuts(runner, model_folders[name], CONFIGS[name].vocab_size, None, monkeypatch)


@pytest.mark.parametrize("dtype", ["float8_e4m3fn", "int8"])
def test_a_layer_that_reads_another_layers_8bit_cache(dtype, tmp_path, monkeypatch):
    """Layer 0 runs twice with a cache each time, a last layer without keys and values of its own reads layer 1's."""
    from pulse_infer_b200.config import Qwen3Config, register_architecture
    from pulse_infer_b200.engine import build_runner
    from pulse_infer_b200.models.qwen3 import build_qwen3_spec
    from pulse_infer_b200.models.spec import ScheduleEntry
    from pulse_infer_b200.weights import write_random_model
    need_gpu()

    @dataclasses.dataclass(frozen=True)
    class ReaderConfig(Qwen3Config):
        pass

    def build_spec(config):
        spec = build_qwen3_spec(config)
        layers = list(spec.layers)
        layers[2] = dataclasses.replace(layers[2], mixer=dataclasses.replace(layers[2].mixer, params={**layers[2].mixer.params, "writes_cache": False}))
        return dataclasses.replace(spec, layers=tuple(layers),
                                   order=(ScheduleEntry(0, 0), ScheduleEntry(1, 1), ScheduleEntry(0, 2), ScheduleEntry(2, 1)))

    register_architecture("ReaderForCausalLM", ReaderConfig, build_spec, replace=True)
    fields = {f.name: getattr(CONFIGS["E"], f.name) for f in dataclasses.fields(CONFIGS["E"])}
    cfg = ReaderConfig(**{**fields, "architecture": "ReaderForCausalLM", "num_hidden_layers": 3})
    folder = write_random_model(cfg, 9, str(tmp_path / "reader"), dtype="bfloat16")
    for graphs in (False, True):
        runner = build_runner(folder, dtype="bfloat16", device="cuda:0", page_size=16, num_pages=64, max_requests=4,
                              max_tokens_per_request=512, cache_dtype=dtype, use_cuda_graphs=graphs)
        _run_cuts(runner, folder, cfg.vocab_size, [(0, 0), (1, 1), (0, 2), (2, 1)], monkeypatch)
