"""Engines with an 8-bit cache: logits against the plain implementation on encoded keys and values, every way of cutting
requests into steps, recorded steps against launched ones, generation, preemption, the command line; and what is refused."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_model
from cache8_util import BLOCK, encode, exponent
from gpu_util import need_gpu
from helpers import load_plain, random_tokens
from tiny_configs import CONFIGS

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"float8_e4m3fn": torch.float8_e4m3fn, "int8": torch.int8}
# Fraction of the largest |logit|.  With bfloat16 pages 2e-2 is allowed for keys and values that are off by about one
# bfloat16 half step, dev = 2^-8 of themselves.  Encoded, two values that far apart fall to different codes with
# probability dev / step and are then a step apart: sqrt(dev * step) on average.  e4m3, step 2^-3 of the value: 2^-5.5, six
# times dev, and nine with the error of the encoding's own slope allowed for.  int8, step about 1/90 of the block's largest
# magnitude, dev 2^-8 of a third of it: three times dev; the extra encodings of a block that grows token by token, each off
# by step / sqrt(12), add as much again: five.
TOL = {"float8_e4m3fn": 9 * 2e-2, "int8": 5 * 2e-2}


def _runner(folder, cache_dtype, **kw):
    from pulse_infer_b200.engine import build_runner
    args = dict(dtype="bfloat16", device="cuda:0", page_size=16, num_pages=96, max_requests=4, max_tokens_per_request=512,
                cache_dtype=cache_dtype)
    args.update(kw)
    return build_runner(folder, **args)


def _encoded(x, dtype):
    """x [T, heads, d] as the pages hold it: blocks of 16 tokens."""
    out = np.empty_like(x)
    for lo in range(0, x.shape[0], BLOCK):
        for h in range(x.shape[1]):
            part = torch.tensor(x[lo:lo + BLOCK, h])
            e = exponent(part.abs().max().item(), dtype)
            out[lo:lo + BLOCK, h] = (encode(part * 2.0 ** -e, dtype) * 2.0 ** e).numpy()
    return out


@pytest.fixture
def plain_8bit(monkeypatch):
    """The plain implementation's forward over encoded keys and values."""
    real = plain_model.layer_keys_values

    def run(folder, dtype, tokens):
        cfg, w = load_plain(folder)
        monkeypatch.setattr(plain_model, "layer_keys_values",
                            lambda *a, **k: tuple(_encoded(x, DTYPES[dtype]) for x in real(*a, **k)))
        try:
            return plain_model.forward(cfg, w, tokens)
        finally:
            monkeypatch.setattr(plain_model, "layer_keys_values", real)
    return run


def _check(got, want, scale, dtype, what):
    err = np.abs(got.detach().cpu().double().numpy() - want).max()
    assert err <= TOL[dtype] * scale, f"{what}: off by {err:.3e} of {scale:.3e}"
    return err / scale


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("name,page", [("D", 16), ("E", 16), ("E", 64), ("D", 128)])
def test_every_cut_against_the_plain_implementation(name, page, dtype, model_folders, plain_8bit):
    from pulse_infer_b200.engine import Segment
    need_gpu()
    folder, cfg = model_folders[name], CONFIGS[name]
    for graphs in (False, True):
        runner = _runner(folder, dtype, page_size=page, use_cuda_graphs=graphs)
        for seed, n in ((1, 200), (2, 33), (3, 1)):
            toks = random_tokens(seed, n, cfg.vocab_size)
            want = plain_8bit(folder, dtype, toks)
            scale = np.abs(want).max()
            runner.open("w")
            _check(runner.step([Segment("w", toks, list(range(n)))]), want, scale, dtype, f"whole n={n}")
            runner.close("w")
            head = max(0, n - 40)
            runner.open("d")
            if head:
                _check(runner.step([Segment("d", toks[:head], [head - 1])]), want[head - 1:head], scale, dtype, "head")
            for i in range(head, n):
                _check(runner.step([Segment("d", [toks[i]], [0])]), want[i:i + 1], scale, dtype, f"token {i}")
            runner.close("d")
            # portions beside another request that decodes
            runner.open("p"); runner.open("x")
            runner.step([Segment("x", random_tokens(9, 21, cfg.vocab_size), [])])
            at, k, sizes = 0, 0, [7, 2, 13, 1, 5, 31, 2, 70]
            while at < n:
                c = min(sizes[k % len(sizes)], n - at)
                k += 1
                got = runner.step([Segment("x", [k % cfg.vocab_size], []), Segment("p", toks[at:at + c], list(range(c)))])
                _check(got, want[at:at + c], scale, dtype, f"portion [{at}, {at + c})")
                at += c
            runner.check_device_errors()
            runner.close("p"); runner.close("x")
            runner.cache.check_invariants()


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("name", ["D", "E"])
def test_recorded_steps_equal_launched_ones(name, dtype, model_folders):
    """The same kernels on the same pages: bit for bit, over batches that shrink and grow and cross pages."""
    from pulse_infer_b200.engine import Segment
    need_gpu()
    folder, cfg = model_folders[name], CONFIGS[name]
    logits = []
    for graphs in (False, True):
        runner = _runner(folder, dtype, use_cuda_graphs=graphs)
        rows = []
        for i, n in enumerate((30, 5, 160)):
            runner.open(i)
            rows.append(runner.step([Segment(i, random_tokens(i, n, cfg.vocab_size), [n - 1])]).clone())
        for step in range(40):
            batch = [i for i in range(3) if (step // 7 + i) % 3 != 0]
            rows.append(runner.step([Segment(i, [(step * 31 + i * 7) % cfg.vocab_size], [0]) for i in batch]).clone())
        runner.check_device_errors()
        assert not graphs or runner.graphs.recordings > 0
        logits.append(torch.cat(rows))
    assert torch.equal(logits[0], logits[1])


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_generation_lookahead_preemption_and_pages(dtype, model_folders):
    """Greedy generation gives the same tokens with recorded steps, lookahead and both off; all pages come back; a pool too
    small for all requests preempts and still finishes."""
    need_gpu()
    from pulse_infer_b200 import Engine
    folder, cfg = model_folders["E"], CONFIGS["E"]
    prompts = [random_tokens(s, n, cfg.vocab_size) for s, n in ((1, 3), (2, 40), (3, 130))]
    results = []
    for kw in (dict(), dict(lookahead=False), dict(lookahead=False, use_cuda_graphs=False)):
        engine = Engine(folder, page_size=16, num_pages=40, max_batch_size=3, chunk_size=64, cache_dtype=dtype, **kw)
        results.append(engine.generate(prompts, max_new_tokens=20, ignore_eos=True))
        engine.runner.check_device_errors()
        assert list(engine.get_stats().free_pages) == [40]
    assert results[0] == results[1] == results[2] and all(len(r) == 20 for r in results[0])
    engine = Engine(folder, page_size=16, num_pages=12, max_batch_size=3, chunk_size=64, max_tokens_per_request=192, cache_dtype=dtype)
    out = engine.generate([random_tokens(s, 50, cfg.vocab_size) for s in range(4)], max_new_tokens=40, ignore_eos=True)
    assert all(len(r) == 40 for r in out) and list(engine.get_stats().free_pages) == [12]
    assert engine.get_stats().num_preemptions > 0


def test_a_pool_of_a_size_holds_twice_the_tokens(model_folders):
    need_gpu()
    sizes = {}
    for cache in (None, "float8_e4m3fn", "int8"):
        runner = _runner(model_folders["E"], cache, num_pages=None, kv_bytes=8 << 20)
        sizes[cache] = runner.cache.num_pages
        for g in runner.cache.groups:
            held = [g.pool] if g.pool is not None else [t for pools in g.pools_8bit for t in pools]
            assert sum(t.numel() * t.element_size() for t in held) <= 8 << 20
    assert sizes["int8"] == sizes["float8_e4m3fn"] >= int(1.9 * sizes[None])


def test_what_an_8bit_cache_refuses(model_folders):
    need_gpu()
    from pulse_infer_b200 import Engine
    for kw, words in ((dict(dtype="float32"), "bfloat16"), (dict(attention_impl="simple"), "bfloat16"), (dict(page_size=8), "page size"),
                      (dict(cache_dtype="float16"), "cache_dtype")):
        with pytest.raises(ValueError, match=words):
            Engine(model_folders["E"], **{**dict(num_pages=8, cache_dtype="int8"), **kw})
    with pytest.raises(ValueError, match="head size 48"):
        Engine(model_folders["C"], num_pages=8, cache_dtype="int8")


def test_more_requests_than_a_decode_launch_takes(model_folders):
    """1,030 requests decoding in one step, against the same in two steps of 515 (of which each is one launch a layer)."""
    from pulse_infer_b200.engine import Segment
    need_gpu()
    vocab, R, logits = CONFIGS["D"].vocab_size, 1030, []
    for cuts in ([R], [R // 2, R]):
        runner = _runner(model_folders["D"], "int8", num_pages=R, max_requests=R, max_tokens_per_request=16)
        for r in range(R):
            runner.open(r)
        for lo in range(0, R, 206):
            runner.step([Segment(r, [(7 * r) % vocab, (11 * r + 3) % vocab, r % 5], []) for r in range(lo, lo + 206)])
        rows, lo = [], 0
        for hi in cuts:
            rows.append(runner.step([Segment(r, [(13 * r) % vocab], [0]) for r in range(lo, hi)]).double().cpu())
            lo = hi
        runner.check_device_errors()
        logits.append(torch.cat(rows))
    _check(logits[0], logits[1].numpy(), logits[1].abs().max().item(), "int8", "one step against two")
    assert (logits[1][:515] - logits[1][515:]).abs().max() > 0.5 * logits[1].abs().max()       # requests do differ


def test_an_8bit_cache_for_more_requests_than_page_maps_take(model_folders):
    need_gpu()
    from pulse_infer_b200 import Engine
    with pytest.raises(ValueError, match="at most 4096 requests"):
        Engine(model_folders["E"], num_pages=8, cache_dtype="int8", max_batch_size=4097)


def test_command_line_with_an_8bit_cache(model_folders):
    need_gpu()
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "qwen3_continuous_batch_demo"), model_folders["E"], "--prompt-len", "40",
                          "--prompt-len", "9", "--max-new-tokens", "6", "--cache-dtype", "float8_e4m3fn", "--ignore-eos"],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
    recs = [json.loads(l) for l in out.stdout.splitlines() if l.startswith("{")]
    assert [len(r["generated"]) for r in recs] == [6, 6]
    out = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "qwen3_infer"), model_folders["D"], "--prompt-len", "40", "--cache-dtype", "int8",
                          "--max-new-tokens", "6", "--ignore-eos", "--repetition-penalty", "1.2", "--frequency-penalty", "0.3"],
                         capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-2000:]
