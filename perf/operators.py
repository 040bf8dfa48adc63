"""What is measured of the operators around the 8-bit paged cache and of the logit rules: the cases, their inputs, the
operators in plain torch operations, and their values in 64 bits.

The operators (``own``: as the framework's entry points; otherwise plain):

* ``maps``    block tables and slot maps of a step, from the lengths of its requests;
* ``write``   per-head norm and rotation of queries and keys, keys and values quantised into their 8-bit pages; the pages
              that were touched are read back as bfloat16 (their 8-bit values times a power of two are exact there);
* ``decode``  one query token per request over the 8-bit pages;
* ``prompt``  portions of prompts over the 8-bit pages (the page maps included);
* ``rules``   penalties for repeated tokens, biases and bit masks on logits.

The 8-bit pages: a block is 16 tokens of one key/value head.  Keys [pages, heads, page, size], values transposed within a
block [pages, heads, page / 16, size, 16]; per block a scale 2^e with the smallest e for which the block's largest
magnitude is at most 448 (e4m3) or 127 (int8) times 2^e, e within [-40, 40].  A block that grows keeps or raises its
scale; what it holds is then encoded again.  Keys are rounded to bfloat16 before they are encoded.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

BLOCK = 16
E_MIN, E_MAX = -40, 40
EPS = 1e-6
THETA = 1e6
VOCAB = 151936


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed() -> list:
    model = {"nq": 32, "nkv": 8, "d": 128, "page": 16, "window": 0}
    return [
        # a decode step of eight requests: the smallest call, launch latency
        {"name": "maps_decode_8", "op": "maps", "requests": 8, "singles": 8, "ctx_lo": 4000, "ctx_hi": 4095, "new_lo": 1,
         "new_hi": 1, "page": 16, "window": 0, "min_tokens": 2, "mix": 1},
        # a full serving step: portions of prompts beside decoding requests, contexts to 32k, every page listed
        {"name": "maps_serving_64", "op": "maps", "requests": 64, "singles": 56, "ctx_lo": 0, "ctx_hi": 32000, "new_lo": 100,
         "new_hi": 512, "page": 16, "window": 0, "min_tokens": 1, "mix": 2},
        # one token each of eight decoding requests
        {"name": "write_decode_8", "op": "write", "dtype": "e4m3", "requests": 8, "singles": 8, "ctx_lo": 4000, "ctx_hi": 4095,
         "new_lo": 1, "new_hi": 1, "adjacent": True, "mix": 3, **model},
        # two portions of about 1,024 tokens, the second starting inside a block
        {"name": "write_prompt_2048", "op": "write", "dtype": "int8", "requests": 2, "singles": 0, "ctx_lo": 0, "ctx_hi": 1003,
         "new_lo": 1019, "new_hi": 1029, "adjacent": True, "mix": 4, **model},
        # the benchmark's decode step: batch 8 at context 4,096
        {"name": "decode_8x4096", "op": "decode", "dtype": "e4m3", "requests": 8, "singles": 8, "ctx_lo": 4000, "ctx_hi": 4095,
         "new_lo": 1, "new_hi": 1, "mix": 5, **model},
        # one request with a long context
        {"name": "decode_1x32k", "op": "decode", "dtype": "int8", "requests": 1, "singles": 1, "ctx_lo": 32767, "ctx_hi": 32767,
         "new_lo": 1, "new_hi": 1, "mix": 6, **model},
        # a large ragged batch, five query heads per key/value head
        {"name": "decode_64_ragged", "op": "decode", "dtype": "e4m3", "requests": 64, "singles": 64, "ctx_lo": 130,
         "ctx_hi": 8190, "new_lo": 1, "new_hi": 1, "mix": 7, **model, "nq": 40},
        # few short contexts in a window, head size 64, as many key/value heads as query heads
        {"name": "decode_3_short_d64", "op": "decode", "dtype": "int8", "requests": 3, "singles": 3, "ctx_lo": 0, "ctx_hi": 300,
         "new_lo": 1, "new_hi": 1, "mix": 8, "nq": 6, "nkv": 6, "d": 64, "page": 32, "window": 130},
        # a whole prompt of about 2,048 tokens
        {"name": "prompt_2048", "op": "prompt", "dtype": "e4m3", "requests": 1, "singles": 0, "ctx_lo": 0, "ctx_hi": 0,
         "new_lo": 2039, "new_hi": 2039, "mix": 9, **model},
        # a short portion behind a long context
        {"name": "prompt_128_behind_16k", "op": "prompt", "dtype": "int8", "requests": 1, "singles": 0, "ctx_lo": 16384,
         "ctx_hi": 16384, "new_lo": 128, "new_hi": 128, "mix": 10, **model},
        # single-stream generation with penalties only
        {"name": "rules_1", "op": "rules", "rows": 1, "vocab": VOCAB, "history_lo": 4000, "history_hi": 4000, "biases": 0,
         "masks": False, "mix": 11},
        # a serving step with everything: penalties, biases, a grammar mask for most rows
        {"name": "rules_64", "op": "rules", "rows": 64, "vocab": VOCAB, "history_lo": 100, "history_hi": 8000, "biases": 300,
         "masks": True, "mix": 12},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["maps", "write", "decode", "decode", "prompt", "rules"])
    mix = rng.randrange(1 << 30)
    if op == "rules":
        lo = _log_int(rng, 1, 4000)
        return {"op": op, "rows": _log_int(rng, 1, 64), "vocab": _log_int(rng, 500, VOCAB), "history_lo": lo,
                "history_hi": rng.randint(lo, 8000), "biases": rng.choice([0, _log_int(rng, 1, 300)]),
                "masks": rng.random() < 0.5, "mix": mix}
    case = {"op": op, "page": rng.choice([16, 32, 64]), "window": rng.choice([0, 0, _log_int(rng, 1, 3000)]), "mix": mix}
    if op == "maps":
        requests = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, 500)
        return {**case, "requests": requests, "singles": rng.randint(0, requests), "ctx_lo": 0, "ctx_hi": _log_int(rng, 1, 32000),
                "new_lo": 1, "new_hi": new, "min_tokens": rng.choice([1, 2])}
    case["dtype"] = rng.choice(["e4m3", "int8"])
    case["d"] = rng.choice([64, 128, 128])
    case["nkv"] = rng.choice([1, 2, 4, 8])
    case["nq"] = case["nkv"] * rng.choice([1, 2, 4, 5, 8])
    if op == "write":
        requests = _log_int(rng, 1, 16)
        new = _log_int(rng, 1, max(1, 2000 // requests))
        case.pop("window")
        return {**case, "window": 0, "requests": requests, "singles": rng.randint(0, requests), "ctx_lo": 0,
                "ctx_hi": _log_int(rng, 1, 2000), "new_lo": 1, "new_hi": new, "adjacent": rng.random() < 0.7}
    if op == "decode":
        requests = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 1, min(32768, 270000 // requests))
        return {**case, "requests": requests, "singles": requests, "ctx_lo": rng.randint(0, ctx), "ctx_hi": ctx, "new_lo": 1,
                "new_hi": 1}
    requests = _log_int(rng, 1, 4)
    new = _log_int(rng, 2, max(2, 1500 // requests))
    ctx = _log_int(rng, 1, max(1, min(12000, 3_000_000 // (new * requests))))
    return {**case, "requests": requests, "singles": 0, "ctx_lo": 0, "ctx_hi": ctx, "new_lo": max(2, new // 2), "new_hi": new}


# ---- shapes of a batch: from the case alone ---------------------------------------------------------------------------
def _batch(case: dict) -> tuple:
    """(start, new tokens) of every request."""
    rng = random.Random(case["mix"])
    starts = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["requests"])]
    news = [1 if i < case["singles"] else rng.randint(case["new_lo"], case["new_hi"]) for i in range(case["requests"])]
    order = list(range(case["requests"]))
    rng.shuffle(order)
    return [starts[i] for i in order], [news[i] for i in order]


def _histories(case: dict) -> list:
    rng = random.Random(case["mix"])
    return [rng.randint(case["history_lo"], case["history_hi"]) for _ in range(case["rows"])]


def _first_page(start: int, window: int, page: int) -> int:
    return max(0, start - window + 1) // page if window else 0


def _listed_pages(case: dict, starts: list, news: list, min_tokens: int) -> int:
    page, window = case["page"], case["window"]
    return sum((a + n - 1) // page - _first_page(a, window, page) + 1 for a, n in zip(starts, news) if n >= min_tokens)


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _exponent(amax: torch.Tensor, dtype: str) -> torch.Tensor:
    """The smallest e with amax <= qmax 2^e, within [E_MIN, E_MAX]."""
    m, e = torch.frexp(amax.float())                     # amax = m 2^e, m in [0.5, 1)
    top, shift = (0.875, 9) if dtype == "e4m3" else (0.9921875, 7)
    return (e - shift + (m > top)).masked_fill(amax == 0, E_MIN).masked_fill(torch.isinf(amax), E_MAX).clamp(E_MIN, E_MAX)


def _encode(x: torch.Tensor, dtype: str) -> torch.Tensor:
    """float32, already divided by the scale -> 8 bits, to nearest even."""
    if dtype == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return x.round().clamp(-127.0, 127.0).to(torch.int8)


def _take(pool: torch.Tensor, pages: torch.Tensor) -> torch.Tensor:
    """pool[pages] in float32 (8-bit floats are indexed as bytes)."""
    return pool.view(torch.uint8)[pages].view(pool.dtype).float()


def _rope_tables(positions: torch.Tensor, d: int) -> tuple:
    div = THETA ** (torch.arange(0, d, 2, dtype=torch.float64, device=positions.device) / d)
    angle = positions.double()[:, None] / div
    return angle.cos().float(), angle.sin().float()


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rnd = random.Random(seed)
    s = {"case": case}
    if case["op"] == "rules":
        return _prepare_rules(case, seed, g, dev, s)
    starts, news = _batch(case)
    R, P = case["requests"], case["page"]
    per = [(a + n + P - 1) // P for a, n in zip(starts, news)]
    width, total = max(per) + 2, sum(per) + 3
    perm = np.random.RandomState(seed % (1 << 31)).permutation(total)
    slots = rnd.sample(range(R + 2), R)
    table = np.full((R + 2, width), -1, dtype=np.int32)
    at = 0
    for slot, n in zip(slots, per):
        table[slot, :n] = perm[at:at + n]
        at += n

    def i32(v):
        return torch.tensor(np.asarray(v, dtype=np.int32), device=dev)
    T = sum(news)
    s.update(block_table=i32(table), seg_slot=i32(slots), seg_start=i32(starts), seg_len=i32(news), num_tokens=T,
             seg_off=i32(np.concatenate([[0], np.cumsum(news)[:-1]])), max_len=max(a + n for a, n in zip(starts, news)),
             max_new=max(news))
    if case["op"] == "maps":
        s["listed"] = _listed_pages(case, starts, news, case["min_tokens"])
        return s
    nq, nkv, d, dtype = case["nq"], case["nkv"], case["d"], case["dtype"]
    # pages as a run leaves them: every block encoded from keys (channels of unequal size) and values (tokens of unequal
    # size); pages of no request hold what an earlier one left there
    sub = P // BLOCK
    channel = 1 + 0.3 * torch.randn(d, generator=g, device=dev)
    pools = []
    for which in range(2):
        pool = torch.empty((total, nkv, P, d), dtype=torch.float8_e4m3fn if dtype == "e4m3" else torch.int8, device=dev)
        scales = torch.empty((total, nkv, sub), dtype=torch.float32, device=dev)
        step = max(1, (1 << 26) // (nkv * P * d))
        for lo in range(0, total, step):
            n = min(step, total - lo)
            x = torch.randn((n, nkv, sub, BLOCK, d), generator=g, device=dev)
            x *= channel if which == 0 else torch.exp(0.7 * torch.randn((n, nkv, sub, BLOCK, 1), generator=g, device=dev))
            e = _exponent(x.abs().amax((-1, -2)), dtype)
            scales[lo:lo + n] = torch.exp2(e.float())
            q = _encode(x * torch.exp2(-e.float())[..., None, None], dtype)
            pool[lo:lo + n] = q.view(n, nkv, P, d)
        if which == 1:
            pool = pool.view(torch.uint8).view(total, nkv, sub, BLOCK, d).transpose(3, 4).contiguous().view(pool.dtype)
        pools += [pool, scales]
    s.update(kcache=pools[0], kscale=pools[1], vcache=pools[2], vscale=pools[3])
    if case["op"] == "write":
        positions = np.concatenate([np.arange(a, a + n) for a, n in zip(starts, news)])
        slot_of = np.repeat(slots, news)
        slot_map = table[slot_of, positions // P].astype(np.int64) * P + positions % P
        s["slot_map"] = torch.tensor(slot_map, device=dev)
        s["touched"] = i32(np.unique(slot_map // P))
        x = torch.randn((T, nq + 2 * nkv, d), generator=g, device=dev)
        x[:, nq + nkv:] *= torch.exp(0.7 * torch.randn((T, nkv, 1), generator=g, device=dev))
        s["qkv"] = x.view(T, -1).to(torch.bfloat16)
        s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(torch.bfloat16)
        s["k_weight"] = channel.to(torch.bfloat16)
        s["cos"], s["sin"] = _rope_tables(torch.tensor(positions, device=dev), d)
        s["errors"] = torch.zeros(1, dtype=torch.int32, device=dev)
        return s
    s["q"] = (2 * torch.randn((T, nq * d), generator=g, device=dev)).to(torch.bfloat16)
    s["listed"] = _listed_pages(case, starts, news, 1)
    if own and case["op"] == "decode":
        from pulse_infer_b200 import ops
        s["workspace"] = ops.attention_decode_workspace(d, dev)
    return s


def _prepare_rules(case, seed, g, dev, s):
    n, V = case["rows"], case["vocab"]
    lens = _histories(case)
    r = np.random.RandomState(seed % (1 << 31))
    s["logits"] = 3 * torch.randn((n, V), generator=g, device=dev)
    # tokens as text has them: a few ids make up most of a history
    ids = [np.minimum((V * r.rand(L) ** 3).astype(np.int64), V - 1) for L in lens]
    s["history"] = torch.tensor(np.concatenate(ids).astype(np.int32), device=dev)
    s["history_off"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), device=dev)
    s["prompt_len"] = torch.tensor([int(r.randint(0, L + 1)) for L in lens], dtype=torch.int32, device=dev)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=dev)  # noqa: E731
    s["repetition"] = f(r.choice([1.0, 1.05, 1.2, 1.3], n))
    s["frequency"] = f(r.choice([0.0, 0.2, 0.5], n))
    s["presence"] = f(r.choice([0.0, 0.4, 1.5], n))
    if case["biases"]:
        count = [int(r.randint(0, min(case["biases"], V) + 1)) for _ in range(n)]
        s["bias_off"] = torch.tensor(np.concatenate([[0], np.cumsum(count)]).astype(np.int32), device=dev)
        s["bias_tokens"] = torch.tensor(np.concatenate([r.permutation(V)[:c] for c in count]).astype(np.int32), device=dev)
        s["bias_values"] = f(r.uniform(-5, 5, sum(count)))
    if case["masks"]:
        rows = max(1, n - n // 4)
        words = r.randint(-2 ** 31, 2 ** 31, (rows, (V + 31) // 32), dtype=np.int64)
        s["mask"] = torch.tensor(words.astype(np.int32), device=dev)
        s["mask_row"] = torch.tensor(np.where(np.arange(n) < rows, np.arange(n), -1).astype(np.int32), device=dev)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------
def run(state: dict):
    case = state["case"]
    if own:
        return _OWN[case["op"]](state, case)
    return _PLAIN[case["op"]](state, case)


def _own_maps(s, c):
    from pulse_infer_b200 import ops
    m = ops.page_maps(s["block_table"], s["seg_slot"], s["seg_start"], s["seg_len"], c["page"], s["num_tokens"],
                      num_listed_pages=s["listed"], window=c["window"] or None, min_tokens=c["min_tokens"])
    return {"seg_off": m.seg_off, "positions": m.positions, "token_seg": m.token_seg, "slot_map": m.slot_map,
            "page_off": m.page_off, "page_list": m.page_list, "table": m.table}


def _own_write(s, c):
    from pulse_infer_b200 import ops
    q = ops.qk_norm_rope_write_8bit(s["qkv"], s["q_weight"], s["k_weight"], EPS, s["cos"], s["sin"], c["adjacent"], s["kcache"],
                                    s["vcache"], s["kscale"], s["vscale"], s["slot_map"], c["nq"], c["nkv"], c["d"], s["errors"])
    keys, values = ops.pages_8bit_to_bf16(s["kcache"], s["vcache"], s["kscale"], s["vscale"], s["touched"])
    return {"q": q, "keys": keys, "values": values}


def _own_decode(s, c):
    from pulse_infer_b200 import ops
    return ops.attention_decode_8bit(s["q"], c["nq"] * c["d"], s["kcache"], s["vcache"], s["kscale"], s["vscale"],
                                     s["block_table"], s["seg_off"], s["seg_slot"], s["seg_start"], s["seg_len"],
                                     s["num_tokens"], c["requests"], c["nq"], c["nkv"], c["d"], c["window"] or None,
                                     1.0 / math.sqrt(c["d"]), workspace=s["workspace"])


def _own_prompt(s, c):
    from pulse_infer_b200 import ops
    m = ops.page_maps(s["block_table"], s["seg_slot"], s["seg_start"], s["seg_len"], c["page"], s["num_tokens"],
                      num_listed_pages=s["listed"], window=c["window"] or None, min_tokens=2)
    starts, news = _batch(c)
    return ops.attention_prompt_8bit(s["q"], c["nq"] * c["d"], s["kcache"], s["vcache"], s["kscale"], s["vscale"], m,
                                     s["seg_start"], s["seg_len"], list(zip(starts, news)), s["num_tokens"], c["nq"], c["nkv"],
                                     c["d"], c["window"] or None, 1.0 / math.sqrt(c["d"]))


def _own_rules(s, c):
    from pulse_infer_b200 import ops
    return ops.logit_rules(s["logits"], s["history"], s["history_off"], s["prompt_len"], s["repetition"], s["frequency"],
                           s["presence"], bias_off=s.get("bias_off"), bias_tokens=s.get("bias_tokens"),
                           bias_values=s.get("bias_values"), mask=s.get("mask"), mask_row=s.get("mask_row"))


def _plain_maps(s, c):
    P, W, T, N = c["page"], s["block_table"].shape[1], s["num_tokens"], s["listed"]
    dev = s["block_table"].device
    start, length = s["seg_start"].long(), s["seg_len"].long()
    rows = s["block_table"][s["seg_slot"].long()].long()
    zero = torch.zeros(1, dtype=torch.long, device=dev)
    seg_off = torch.cat([zero, length.cumsum(0)])
    t = torch.arange(T, device=dev)
    token_seg = torch.searchsorted(seg_off[1:], t, right=True)
    positions = start[token_seg] + t - seg_off[token_seg]
    page = rows[token_seg, positions // P]
    slot_map = torch.where(page >= 0, page * P + positions % P, -1)
    first = (start - c["window"] + 1).clamp(min=0) // P if c["window"] else torch.zeros_like(start)
    last = (start + length - 1) // P
    count = torch.where(length >= c["min_tokens"], last - first + 1, 0)
    page_off = torch.cat([zero, count.cumsum(0)])
    i = torch.arange(N, device=dev)
    owner = torch.searchsorted(page_off[1:], i, right=True)
    page_list = rows[owner, first[owner] + i - page_off[owner]] if N else zero[:0]
    w = torch.arange(W, device=dev)
    inside = (w >= first[:, None]) & (w < (first + count)[:, None])
    table = torch.where(inside, page_off[:-1, None] + w - first[:, None], -1)
    return {"seg_off": seg_off.int(), "positions": positions.int(), "token_seg": token_seg.int(), "slot_map": slot_map,
            "page_off": page_off.int(), "page_list": page_list.int(), "table": table.int()}


def _norm_rope(x, weight, cos, sin, adjacent):
    """x float32 [T, heads, d]: RMSNorm over d, then rotation of all pairs."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    a, b = (x[..., 0::2], x[..., 1::2]) if adjacent else x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    r0, r1 = a * c - b * s, a * s + b * c
    return torch.stack([r0, r1], -1).flatten(-2) if adjacent else torch.cat([r0, r1], -1)


def _plain_store(pool, scales, x, where, pages, dtype, transposed):
    """x float32 [T, heads, d] into rows ``where`` (slots counted within ``pages``) of the pool, in place."""
    n, (nkv, sub) = pages.numel(), scales.shape[1:]
    d = x.shape[-1]
    old = _take(pool, pages)
    if transposed:
        old = old.transpose(3, 4)
    old = old.reshape(n, nkv, sub, BLOCK, d).permute(0, 2, 1, 3, 4).reshape(n * sub, nkv, BLOCK, d)
    e_old = torch.log2(scales[pages].permute(0, 2, 1).reshape(n * sub, nkv))
    blk, off = where // BLOCK, where % BLOCK
    wide = blk[:, None].expand(-1, nkv)
    amax = torch.zeros((n * sub, nkv), device=x.device).scatter_reduce_(0, wide, x.abs().amax(-1), "amax")
    lowest = torch.full((n * sub,), BLOCK, device=x.device, dtype=torch.long).scatter_reduce_(0, blk, off, "amin")
    touched, began = (lowest < BLOCK)[:, None], (lowest == 0)[:, None]
    e_new = torch.where(touched, torch.maximum(torch.where(began, float(E_MIN), e_old), _exponent(amax, dtype).float()), e_old)
    kept = torch.where(began[..., None, None], 0.0, old * torch.exp2(torch.where(began, 0.0, e_old - e_new))[..., None, None])
    rows = _encode(kept, dtype)
    new = _encode(x * torch.exp2(-e_new)[blk][..., None], dtype)
    raw = rows.view(torch.uint8)
    raw[blk, :, off] = new.view(torch.uint8)
    raw = raw.view(n, sub, nkv, BLOCK, d).permute(0, 2, 1, 3, 4)
    raw = raw.transpose(3, 4) if transposed else raw.reshape(n, nkv, sub * BLOCK, d)
    pool.view(torch.uint8)[pages] = raw
    scales[pages] = torch.exp2(e_new).view(n, sub, nkv).permute(0, 2, 1)


def _plain_dense(pool, scales, pages, transposed):
    """Pages as float32 [..., heads, page, d], scaled."""
    x = _take(pool, pages)
    lead = pages.shape
    nkv, sub = scales.shape[1:]
    x = x.transpose(-1, -2) if transposed else x.unflatten(-2, (sub, BLOCK))
    return (x * scales[pages][..., None, None]).reshape(*lead, nkv, sub * BLOCK, x.shape[-1])


def _plain_write(s, c):
    T, nq, nkv, d, P = s["num_tokens"], c["nq"], c["nkv"], c["d"], c["page"]
    x = s["qkv"].float().view(T, nq + 2 * nkv, d)
    q = _norm_rope(x[:, :nq], s["q_weight"], s["cos"], s["sin"], c["adjacent"]).to(torch.bfloat16)
    k = _norm_rope(x[:, nq:nq + nkv], s["k_weight"], s["cos"], s["sin"], c["adjacent"]).to(torch.bfloat16).float()
    pages = s["touched"].long()
    inverse = torch.zeros(s["kcache"].shape[0], dtype=torch.long, device=x.device)
    inverse[pages] = torch.arange(pages.numel(), device=x.device)
    where = inverse[s["slot_map"] // P] * P + s["slot_map"] % P
    _plain_store(s["kcache"], s["kscale"], k, where, pages, c["dtype"], False)
    _plain_store(s["vcache"], s["vscale"], x[:, nq + nkv:], where, pages, c["dtype"], True)
    return {"q": q.view(T, nq * d), "keys": _plain_dense(s["kcache"], s["kscale"], pages, False).to(torch.bfloat16),
            "values": _plain_dense(s["vcache"], s["vscale"], pages, True).to(torch.bfloat16)}


def _plain_attention(s, c, queries, positions):
    """queries float32 [R, L, nq, d] at ``positions`` [R, L] (-1: none) over the pages; -> [R, L, nq, d]."""
    nkv, d, P = c["nkv"], c["d"], c["page"]
    R, L, nq = queries.shape[:3]
    W = (s["max_len"] + P - 1) // P
    pages = s["block_table"][s["seg_slot"].long(), :W].long().clamp(min=0)
    k = _plain_dense(s["kcache"], s["kscale"], pages, False).transpose(1, 2).reshape(R, nkv, W * P, d)
    v = _plain_dense(s["vcache"], s["vscale"], pages, True).transpose(1, 2).reshape(R, nkv, W * P, d)
    q = queries.view(R, L, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(R, nkv, -1, d)
    scores = (q @ k.transpose(2, 3)).view(R, nkv, nq // nkv, L, W * P) / math.sqrt(d)
    at = torch.arange(W * P, device=q.device)
    seen = at <= positions[..., None]
    if c["window"]:
        seen &= at > positions[..., None] - c["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True)
    out = scores.view(R, nkv, -1, W * P) @ v
    return out.view(R, nkv, nq // nkv, L, d).permute(0, 3, 1, 2, 4).reshape(R, L, nq, d)


def _plain_decode(s, c):
    R, nq, d = c["requests"], c["nq"], c["d"]
    out = _plain_attention(s, c, s["q"].float().view(R, 1, nq, d), s["seg_start"].long()[:, None])
    return out.view(R, nq * d).to(torch.bfloat16)


def _plain_prompt(s, c):
    R, nq, d, L, T = c["requests"], c["nq"], c["d"], s["max_new"], s["num_tokens"]
    i = torch.arange(L, device=s["q"].device)
    row = (s["seg_off"].long()[:, None] + i).clamp(max=T - 1)
    out = _plain_attention(s, c, s["q"].float().view(T, nq, d)[row], s["seg_start"].long()[:, None] + i)
    ends = s["seg_off"].long() + s["seg_len"].long()
    t = torch.arange(T, device=i.device)
    seg = torch.searchsorted(ends, t, right=True)
    return out[seg, t - s["seg_off"].long()[seg]].view(T, nq * d).to(torch.bfloat16)


def _plain_rules(s, c):
    x = s["logits"]
    n, V = x.shape
    h = torch.arange(s["history"].numel(), device=x.device)
    row = torch.searchsorted(s["history_off"].long()[1:], h, right=True)
    generated = (h - s["history_off"].long()[row] >= s["prompt_len"].long()[row]).float()
    token = row * V + s["history"].long()
    count = torch.zeros(n * V, device=x.device).index_add_(0, token, generated).view(n, V)
    seen = torch.zeros(n * V, device=x.device).index_fill_(0, token, 1.0).view(n, V)
    rep = torch.where(seen > 0, s["repetition"][:, None], 1.0)
    x = torch.where(x > 0, x / rep, x * rep) - s["frequency"][:, None] * count - s["presence"][:, None] * seen
    if "bias_off" in s:
        b = torch.arange(s["bias_tokens"].numel(), device=x.device)
        row = torch.searchsorted(s["bias_off"].long()[1:], b, right=True)
        x = x.view(-1).index_add(0, row * V + s["bias_tokens"].long(), s["bias_values"]).view(n, V)
    if "mask" in s:
        words = s["mask"][s["mask_row"].long().clamp(min=0)]
        allowed = ((words[..., None] >> torch.arange(32, device=x.device)) & 1).view(n, -1)[:, :V] != 0
        x = torch.where(allowed | (s["mask_row"] < 0)[:, None], x, -math.inf)
    return x


_OWN = {"maps": _own_maps, "write": _own_write, "decode": _own_decode, "prompt": _own_prompt, "rules": _own_rules}
_PLAIN = {"maps": _plain_maps, "write": _plain_write, "decode": _plain_decode, "prompt": _plain_prompt, "rules": _plain_rules}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case: dict) -> dict:
    if case["op"] == "rules":
        n, V = case["rows"], case["vocab"]
        masks = 4 * (n - n // 4) * ((V + 31) // 32) if case["masks"] else 0
        return {"bytes": 8 * n * V + 4 * sum(_histories(case)) + masks + 4 * n * case["biases"], "flops": 4 * n * V}
    starts, news = _batch(case)
    T, R, P, window = sum(news), case["requests"], case["page"], case["window"]
    if case["op"] == "maps":
        width = max((a + n + P - 1) // P for a, n in zip(starts, news)) + 2
        pages = _listed_pages(case, starts, news, case["min_tokens"])
        touched = sum((a + n - 1) // P - a // P + 1 for a, n in zip(starts, news))
        return {"bytes": 12 * R + 4 * (touched + pages) + 16 * T + 4 * pages + 4 * R * width + 8 * (R + 1), "flops": 0}
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    if case["op"] == "write":
        blocks = sum((a + n - 1) // BLOCK - a // BLOCK + 1 for a, n in zip(starts, news))
        touched = sum((a + n - 1) // P - a // P + 1 for a, n in zip(starts, news))
        begun = sum(a % BLOCK for a in starts)             # tokens that a touched block held already
        return {"bytes": 2 * T * (nq + 2 * nkv) * d + 2 * T * nq * d + 4 * T * d + 8 * T + 2 * nkv * d * (begun + BLOCK * blocks)
                + 2 * nkv * 4 * 2 * blocks + 2 * touched * nkv * P * d * 3, "flops": 8 * T * (nq + nkv) * d}
    pairs = keys = 0
    for a, n in zip(starts, news):
        first = max(0, a - window + 1) if window else 0
        keys += a + n - first
        if window:
            pairs += sum(min(p + 1, window) for p in range(a, a + n))
        else:
            pairs += n * a + n * (n + 1) // 2
    return {"bytes": 4 * T * nq * d + 2 * nkv * d * keys + 2 * nkv * 4 * (keys // BLOCK + R), "flops": 4 * nq * d * pairs}


# ---- the operators in 64 bits, request by request ---------------------------------------------------------------------
def exact(case: dict, seed: int):
    if case["op"] == "maps":
        return None                                          # whole numbers
    s = prepare(case, seed)
    if case["op"] == "rules":
        return _exact_rules(s, case)
    if case["op"] == "write":
        return _exact_write(s, case)
    nq, nkv, d, P, window = case["nq"], case["nkv"], case["d"], case["page"], case["window"]
    starts, news = _batch(case)
    slots = s["seg_slot"].tolist()
    out, at = [], 0
    for slot, a, n in zip(slots, starts, news):
        held = s["block_table"][slot, :(a + n + P - 1) // P].long()
        k, v = _exact_context(s, held, False)[:, :a + n], _exact_context(s, held, True)[:, :a + n]
        q = s["q"][at:at + n].double().view(n, nq, d)
        pos = torch.arange(a, a + n, device=q.device)[:, None]
        key = torch.arange(a + n, device=q.device)[None]
        hidden = (key > pos) | ((key <= pos - window) if window else torch.zeros_like(key > pos))
        heads = []
        for h in range(nq):
            z = (q[:, h] @ k[h * nkv // nq].T) * d ** -0.5
            z[hidden] = -math.inf
            heads.append(torch.softmax(z, -1) @ v[h * nkv // nq])
        out.append(torch.stack(heads, 1).reshape(n, nq * d))
        at += n
    return torch.cat(out)


def _exact_context(s, held, values):
    """[heads, tokens, d] in 64 bits of the pages ``held``."""
    pool, scale = (s["vcache"], s["vscale"]) if values else (s["kcache"], s["kscale"])
    pages = []
    for block, sc in zip(pool.view(torch.uint8)[held].view(pool.dtype).double().split(64), scale[held].double().split(64)):
        m, nkv, sub = sc.shape
        block = block.mT if values else block.reshape(m, nkv, sub, BLOCK, -1)      # [m, heads, sub, 16, d]
        pages.append((block * sc[..., None, None]).reshape(m, nkv, sub * BLOCK, -1).transpose(0, 1).reshape(nkv, m * sub * BLOCK, -1))
    return torch.cat(pages, 1)


def _exact_write(s, case):
    T, nq, nkv, d, P = s["num_tokens"], case["nq"], case["nkv"], case["d"], case["page"]
    x = s["qkv"].double().cpu().numpy().reshape(T, nq + 2 * nkv, d)
    cos, sin = s["cos"].double().cpu().numpy()[:, None], s["sin"].double().cpu().numpy()[:, None]
    top = 448.0 if case["dtype"] == "e4m3" else 127.0
    first, second = (slice(0, d, 2), slice(1, d, 2)) if case["adjacent"] else (slice(0, d // 2), slice(d // 2, d))

    def turned(part, weight):
        y = part / np.sqrt((part ** 2).mean(-1, keepdims=True) + EPS) * weight.double().cpu().numpy()
        z = np.empty_like(y)
        z[..., first] = y[..., first] * cos - y[..., second] * sin
        z[..., second] = y[..., first] * sin + y[..., second] * cos
        return z

    def coded(v, exponent):
        """What the 8 bits of v / 2^exponent stand for."""
        t = torch.tensor(v * 2.0 ** -exponent)
        if case["dtype"] == "e4m3":                          # spacing 2^(floor(log2) - 3), at least 2^-9
            step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
            return (torch.round(t / step) * step).clamp(-top, top).numpy() * 2.0 ** exponent
        return torch.round(t).clamp(-top, top).numpy() * 2.0 ** exponent

    q = turned(x[:, :nq], s["q_weight"])
    k = torch.tensor(turned(x[:, nq:nq + nkv], s["k_weight"])).to(torch.bfloat16).double().numpy()
    slot_map, pages = s["slot_map"].cpu().numpy(), s["touched"].tolist()
    results = []
    for new, values in ((k, False), (x[:, nq + nkv:], True)):
        scale = (s["vscale"] if values else s["kscale"]).cpu().numpy()
        held = s["touched"].long()
        nowv = _exact_context(s, held, values).view(nkv, len(pages), P, d).transpose(0, 1).cpu().numpy().copy()
        for i, page in enumerate(pages):
            here = np.nonzero(slot_map // P == page)[0]
            for b in sorted(set((slot_map[here] % P // BLOCK).tolist())):
                rows = here[slot_map[here] % P // BLOCK == b]
                off = slot_map[rows] % BLOCK
                for h in range(nkv):
                    high = np.abs(new[rows, h]).max()
                    e = E_MIN if high == 0 else int(np.clip(math.ceil(math.log2(high / top)), E_MIN, E_MAX))
                    block = nowv[i, h, b * BLOCK:(b + 1) * BLOCK]
                    if off.min() == 0:
                        block[:] = 0
                    else:
                        e = max(e, int(round(math.log2(scale[page, h, b]))))
                        block[:] = coded(block, e)
                    block[off] = coded(new[rows, h], e)
        results.append(torch.tensor(nowv))
    return {"q": torch.tensor(q.reshape(T, nq * d)), "keys": results[0], "values": results[1]}


def _exact_rules(s, case):
    x = s["logits"].double().cpu().numpy()
    n, V = x.shape
    history, off = s["history"].cpu().numpy(), s["history_off"].tolist()
    for r in range(n):
        ids = history[off[r]:off[r + 1]]
        generated = ids[int(s["prompt_len"][r]):]
        known = np.unique(ids)
        rep = float(s["repetition"][r])
        x[r, known] = np.where(x[r, known] > 0, x[r, known] / rep, x[r, known] * rep) - float(s["presence"][r])
        x[r] -= float(s["frequency"][r]) * np.bincount(generated, minlength=V)
        if "bias_off" in s:
            lo, hi = int(s["bias_off"][r]), int(s["bias_off"][r + 1])
            x[r, s["bias_tokens"][lo:hi].cpu().numpy()] += s["bias_values"][lo:hi].double().cpu().numpy()
        if "mask" in s and int(s["mask_row"][r]) >= 0:
            words = s["mask"][int(s["mask_row"][r])].cpu().numpy().view(np.uint32)
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:V]
            x[r, bits == 0] = -np.inf
    return torch.tensor(x)
