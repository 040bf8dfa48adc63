"""The entry points around the 8-bit cache and the logit rules refuse tensors that are not on a CUDA device (no fallback)."""
import pytest
import torch


def test_host_tensors_are_refused():
    from pulse_infer_b200 import ops
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    bf = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16)  # noqa: E731
    pools = ops.cache_8bit_pools(2, 2, 16, 64, torch.int8, "cpu")
    assert [tuple(t.shape) for t in pools] == [(2, 2, 16, 64), (2, 2, 1, 64, 16), (2, 2, 1), (2, 2, 1)]
    calls = [lambda: ops.page_maps(i32(2, 3), i32(2), i32(2), i32(2), 16, 2),
             lambda: ops.qk_norm_rope_write_8bit(bf(1, 512), None, None, 1e-6, None, None, True, *pools, torch.zeros(1, dtype=torch.int64), 4, 2, 64, i32(1)),
             lambda: ops.pages_8bit_to_bf16(*pools, i32(1)),
             lambda: ops.attention_decode_8bit(bf(1, 256), 256, *pools, i32(1, 1), i32(1), i32(1), i32(1), i32(1), 1, 1, 4, 2, 64, None, 0.1),
             lambda: ops.logit_rules(torch.zeros(1, 10), i32(0), i32(2), i32(1), torch.ones(1), torch.zeros(1), torch.zeros(1))]
    for call in calls:
        with pytest.raises(ops.KernelError, match="CUDA device only"):
            call()


@pytest.mark.parametrize("bad", [(1, 2, 8, 64, torch.int8), (1, 2, 48, 64, torch.int8), (1, 2, 16, 96, torch.int8), (1, 2, 16, 64, torch.uint8)])
def test_formats_that_do_not_exist(bad):
    from pulse_infer_b200 import ops
    with pytest.raises(ops.KernelError):
        ops.cache_8bit_pools(*bad, "cpu")


def test_histories_beyond_the_counter_are_refused():
    """2^30 entries of one id would carry its count into the bit that says that the id has a bias.  (The launcher refuses
    before it looks at a pointer or at the device.)"""
    import ctypes
    from pulse_infer_b200.ops import kernels
    lib = kernels._lib("sampling")
    launch = lib.pi_logit_rules
    launch.argtypes = kernels._LOGIT_RULES.argtypes
    for history, biases in ((1 << 30, 0), ((1 << 30) + 1, 0), (1 << 40, 0), (0, (1 << 30) + 1)):
        record = kernels._LOGIT_RULES.pack(0, 8, 0, 8, 1, 8, 0, 0, history, 0, 0, 0, 0, 0, 0, 0, biases, 0, 0, 0)
        assert launch(record, None) == -1, (history, biases)
        assert b"beyond the limit" in lib.pi_last_error()


def test_shares_that_32_bits_do_not_hold_are_refused():
    """The number of CTAs is (units + span_min - 1) / span_min: with a span near 2^31 the sum wrapped, and no CTA did anything.
    (Refused before the launcher looks at the device.)"""
    from pulse_infer_b200.ops import cache_8bit, kernels
    lib = kernels._lib("attention_8bit")
    launch = lib.pi_attention_decode_8bit
    launch.argtypes = cache_8bit._DECODE.argtypes
    for span_min, pair_cost in ((2 ** 31 - 1, 2), (1000000001, 2), (2 ** 32 + 2, 2), (-2 ** 32 + 2, 2), (2, 2 ** 32), (0, 2), (2, -1)):
        record = cache_8bit._DECODE.pack(16, 64, 16, 16, 16, 16, cache_8bit.INT8, 1, 16, 1, 1, 16, 16, 16, 16, 16, 16, 16, 16, 148, span_min, pair_cost,
                                         1, 1, 1, 1, 64, 16, 0, 0.1)
        assert launch(record, None) == -1
        assert b"span_min" in lib.pi_last_error(), (span_min, pair_cost, lib.pi_last_error())


def test_page_maps_hand_large_limits_on_as_what_they_mean(monkeypatch):
    from pulse_infer_b200.ops import cache_8bit
    seen = []
    monkeypatch.setattr(cache_8bit, "_on_current_device", lambda tensors: 0)
    monkeypatch.setattr(cache_8bit, "_PAGE_MAPS", lambda device, args: seen.append(args))
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)  # noqa: E731
    for window, min_tokens in ((2 ** 32 + 5, 2 ** 32 + 1), (2 ** 31, 2 ** 31), (7, 2)):
        cache_8bit.page_maps(i32(2, 3), i32(2), i32(2), i32(2), 16, 2, window=window, min_tokens=min_tokens)
    assert [a[10:12] for a in seen] == [(2 ** 31 - 1, 2 ** 31 - 1)] * 2 + [(7, 2)]
