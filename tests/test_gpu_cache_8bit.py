"""The kernels of the 8-bit paged cache against float64, alone and as a step uses them together."""
import math

import numpy as np
import pytest
import torch

import plain_model
from cache8_util import BLOCK, Pools, Sequences, attention_with_bound, encode, exponent, half_step, to_codes
from gpu_util import need_gpu, segments_to_device

pytestmark = pytest.mark.gpu
DTYPES = [torch.float8_e4m3fn, torch.int8]
F16_HALF_STEP, BF16_HALF_STEP = 2.0 ** -11, 2.0 ** -8


def _ops():
    from pulse_infer_b200 import ops
    return ops


# ---- page maps -----------------------------------------------------------------------------------------------------
def plain_maps(table, segs, page, T, N, window, min_tokens):
    """segs: (slot, start, length)."""
    R, W = len(segs), table.shape[1]
    slot_map, positions, token_seg = np.full(T, -1, np.int64), np.zeros(T, np.int64), np.full(T, -1, np.int64)
    page_list, page_tokens = np.full(N, -1, np.int64), np.zeros((N, 2), np.int64)
    tab = np.full((R, W), -1, np.int64)
    seg_off, page_off, t, k = [], [], 0, 0
    for r, (slot, start, n) in enumerate(segs):
        seg_off.append(t); page_off.append(k)
        look = lambda i: int(table[slot, i]) if 0 <= slot < table.shape[0] and 0 <= i < W else -1  # noqa: E731
        for p in range(start, start + n):
            if t < T:
                g = look(p // page)
                slot_map[t] = g * page + p % page if g >= 0 else -1
                positions[t], token_seg[t] = p, r
            t += 1
        if n >= min_tokens and n > 0:
            lo = max(0, start - window + 1) if window else 0
            for i in range(lo // page, (start + n - 1) // page + 1):
                if k < N:
                    page_list[k] = look(i)
                    page_tokens[k] = max(0, lo - i * page), min(page, start + n - i * page)
                    if i < W:
                        tab[r, i] = k
                k += 1
    return dict(slot_map=slot_map, positions=positions, token_seg=token_seg, seg_off=np.array(seg_off + [t]),
                page_off=np.array(page_off + [k]), page_list=page_list, page_tokens=page_tokens, table=tab, rows=np.arange(R))


@pytest.mark.parametrize("page", [16, 32, 1])
@pytest.mark.parametrize("window,min_tokens", [(None, 1), (20, 1), (1, 2), (None, 2), (1000, 3)])
@pytest.mark.parametrize("requests", [1, 7, 300, 1025])
def test_page_maps(page, window, min_tokens, requests):
    dev, ops = need_gpu(), _ops()
    rng = np.random.RandomState(requests * 7 + page)
    slots = requests + 3
    W = (90 + page - 1) // page
    table = rng.permutation(slots * W).reshape(slots, W).astype(np.int32)
    table[rng.rand(slots, W) < 0.05] = -1
    order = rng.permutation(slots)[:requests]
    segs = [(int(s), int(rng.randint(0, 80)), int(rng.choice([0, 1, 1, 2, 9]))) for s in order]
    if requests > 5:
        segs[2] = (segs[2][0], 200, 5)               # positions behind the table
        segs[3] = (slots + 4, 3, 4)                  # a slot that is not there
    total = sum(n for _, _, n in segs)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    pages = int(plain_maps(table, segs, page, total, 10 ** 5, window, min_tokens)["page_off"][-1])
    for T, N in ((total, pages), (total + 5, pages + 3), (max(0, total - 3), max(0, pages - 2)), (0, 0)):
        got = ops.page_maps(i32(table), i32([s for s, _, _ in segs]), i32([a for _, a, _ in segs]), i32([n for _, _, n in segs]),
                            page, T, num_listed_pages=N, window=window, min_tokens=min_tokens)
        for name, want in plain_maps(table, segs, page, T, N, window, min_tokens).items():
            have = getattr(got, name).cpu().numpy()
            assert have.shape == want.shape and np.array_equal(have, want), (name, T, N)


# ---- writing ----------------------------------------------------------------------------------------------------------
def _write(ops, dev, dtype, segs, nq, nkv, d, page, seed, norm=True, rot=1.0, adjacent=True, weight_dtype=torch.bfloat16,
           bump=1.0, special=False):
    """One call over random pools that hold ``start`` tokens of every segment already; everything is checked."""
    g = torch.Generator().manual_seed(seed)
    meta = segments_to_device(segs, dev)
    T = meta["T"]
    per = [(a + n + page - 1) // page for _, a, n in segs]
    pools = Pools(sum(per) + 2, nkv, page, d, dtype, seed)
    perm = torch.randperm(sum(per) + 2, generator=g).tolist()
    table = torch.full((max(s for s, _, _ in segs) + 1, max(per)), -1, dtype=torch.int32)
    for (slot, a, n), count in zip(segs, per):
        for i in range(count):
            table[slot, i] = perm.pop()
            held = min(page, a - i * page)
            if held > 0:
                pools.put(int(table[slot, i]), 0, torch.randn(held, nkv, d, generator=g).double(), torch.randn(held, nkv, d, generator=g).double())
    before = Pools(1, nkv, page, d, dtype)
    before.kcache, before.vcache, before.kscale, before.vscale = (t.clone() for t in (pools.kcache, pools.vcache, pools.kscale, pools.vscale))
    qkv = (bump * torch.randn(T, nq + 2 * nkv, d, generator=g)).to(torch.bfloat16)
    if special:                                       # values only: what is not a number, infinities, zeros, a lone small one
        qkv[0, nq + nkv:, 3] = float("nan")
        qkv[1, nq + nkv:, 5] = float("inf")
        qkv[1, nq + nkv:, 6] = -float("inf")
        qkv[2:, nq + nkv:] = 0
        qkv[2:, nq + nkv:, 1] = 2.0 ** -60
    qw = (1 + 0.2 * torch.randn(d, generator=g)).to(weight_dtype) if norm else None
    kw = (1 + 0.2 * torch.randn(d, generator=g)).to(weight_dtype) if norm else None
    pairs = int(rot * d / 2)
    theta, eps = 10000.0, 1e-5
    cos = sin = None
    if pairs:
        div = torch.tensor([theta ** (2.0 * i / (2 * pairs)) for i in range(pairs)], dtype=torch.float64, device=dev)
        cos, sin = ops.rope_table(meta["positions"], div)
    slot_map = torch.empty(T, dtype=torch.int64)
    t = 0
    for slot, a, n in segs:
        for p in range(a, a + n):
            slot_map[t] = int(table[slot, p // page]) * page + p % page
            t += 1
    dk = pools.on(dev)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    src = qkv.view(T, -1).to(dev)
    move = lambda x: None if x is None else x.to(dev)  # noqa: E731
    q = ops.qk_norm_rope_write_8bit(src, move(qw), move(kw), eps, cos, sin, adjacent, *dk, slot_map.to(dev), nq, nkv, d, err)
    assert int(err.item()) == 0 and torch.equal(src.cpu().view(torch.int16), qkv.view(T, -1).view(torch.int16))
    first = [x.clone() for x in dk]
    q2 = ops.qk_norm_rope_write_8bit(src, move(qw), move(kw), eps, cos, sin, adjacent, *dk, slot_map.to(dev), nq, nkv, d, err)
    for x, y in zip(first, dk):                       # the same step twice does no harm
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    assert torch.equal(q, q2)
    got = Pools(1, nkv, page, d, dtype)
    got.kcache, got.vcache, got.kscale, got.vscale = (x.cpu() for x in dk)
    # ---- what should be there
    x = qkv.double().numpy()
    pos = meta["positions"].cpu().numpy()
    turn = lambda y, w: (lambda z: plain_model.rope(z, pos, theta, 2 * pairs, "adjacent" if adjacent else "half") if pairs else z)(  # noqa: E731
        plain_model.rms_norm(y, w.double().numpy(), eps) if norm else y)
    q_want, k_true = turn(x[:, :nq], qw), torch.tensor(turn(x[:, nq:nq + nkv], kw))
    # two bf16 half steps' room for the rotation's cancellation is not needed: 32-bit arithmetic is off by a few 2^-24 of
    # the row's largest element, the result by half a step of its own
    room = 2.0 ** -20 * np.abs(q_want).max()
    assert (np.abs(q.cpu().double().numpy().reshape(T, nq, d) - q_want) <= BF16_HALF_STEP * np.abs(q_want) + room).all()
    k_room = 2.0 ** -20 * k_true.abs().max()
    v_true = torch.tensor(x[:, nq + nkv:])
    for p in range(pools.pages):
        for b in range(page // BLOCK):
            rows = [i for i in range(T) if slot_map[i] // page == p and slot_map[i] % page // BLOCK == b]
            for h in range(nkv):
                for name, true in (("k", k_true), ("v", v_true)):
                    scale_got, scale_was = (getattr(s, name + "scale")[p, h, b].item() for s in (got, before))
                    pick = (lambda s: s.kcache[p, h, b * BLOCK:(b + 1) * BLOCK]) if name == "k" else (lambda s: s.vcache[p, h, b].T)
                    new, was = pick(got), pick(before)
                    if not rows:                      # untouched, whatever lies there
                        assert torch.equal(new.contiguous().view(torch.uint8), was.contiguous().view(torch.uint8))
                        assert scale_got == scale_was or (math.isnan(scale_got) and math.isnan(scale_was))
                        continue
                    off = [int(slot_map[i]) % BLOCK for i in rows]
                    fresh = true[rows, h]
                    rounded = fresh.to(torch.bfloat16).double()
                    finite = torch.nan_to_num(rounded, nan=0.0, posinf=math.inf, neginf=-math.inf)
                    e = exponent(finite.abs().max().item(), dtype)
                    kept = torch.zeros(BLOCK, d, dtype=torch.float64)
                    if off[0] > 0:
                        e_was = round(math.log2(scale_was))
                        e = max(e, e_was)
                        kept[:off[0]] = encode(was[:off[0]].double() * 2.0 ** (e_was - e), dtype)
                    assert scale_got == 2.0 ** e
                    rest = [i for i in range(BLOCK if off[0] == 0 else off[0]) if i not in off]
                    assert torch.equal(new[rest].double(), kept[rest])
                    have = new[off].double() * 2.0 ** e
                    if name == "v":
                        assert torch.equal(have, encode(rounded * 2.0 ** -e, dtype) * 2.0 ** e)
                    else:
                        assert ((have - fresh).abs() <= half_step(rounded, e, dtype) + BF16_HALF_STEP * fresh.abs() + k_room).all()
    return got


SEGS = [(1, 13, 9), (0, 0, 5), (2, 40, 1), (4, 0, 1), (3, 16, 70), (5, 31, 1)]          # (slot, start, length)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(6, 2, 64, 16), (8, 1, 128, 32), (3, 3, 128, 128), (5, 5, 64, 64), (10, 2, 128, 16)])
def test_write(dtype, nq, nkv, d, page):
    _write(_ops(), need_gpu(), dtype, SEGS, nq, nkv, d, page, seed=nq * d)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm,rot,adjacent,weight_dtype", [(False, 1.0, True, None), (True, 0.5, False, torch.float32),
                                                            (True, 0.0, True, torch.bfloat16), (True, 0.25, True, torch.float32),
                                                            (True, 1.0, False, torch.bfloat16)])
@pytest.mark.parametrize("d", [64, 128])
def test_write_norms_and_rotations(dtype, norm, rot, adjacent, weight_dtype, d):
    _write(_ops(), need_gpu(), dtype, SEGS, 4, 2, d, 16, seed=11, norm=norm, rot=rot, adjacent=adjacent, weight_dtype=weight_dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bump", [1e-3, 40.0, 3e4])
def test_write_blocks_that_grow(dtype, bump):
    """New tokens far above or below what lies in the block: its scale is raised and its codes shifted, or kept."""
    _write(_ops(), need_gpu(), dtype, SEGS, 2, 2, 128, 16, seed=5, bump=bump, norm=False, rot=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_values_that_are_no_numbers(dtype):
    _write(_ops(), need_gpu(), dtype, [(0, 0, 7)], 2, 2, 64, 16, seed=5, special=True)
    _write(_ops(), need_gpu(), dtype, [(0, 3, 7)], 2, 2, 128, 16, seed=6, special=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_tokens_one_by_one_keep_the_formats_range(dtype):
    """A block filled by sixteen steps: the scale is that of the largest token so far, and every token is off by at most
    half a step of each encoding it went through."""
    dev, ops = need_gpu(), _ops()
    nkv, d = 2, 64
    g = torch.Generator().manual_seed(9)
    k, v, ks, vs = ops.cache_8bit_pools(2, nkv, 16, d, dtype, dev)
    sizes = torch.tensor([0.1, 0.1, 0.5, 0.02, 3.0, 3.0, 1.0, 50.0, 2.0, 2.0, 900.0, 1.0, 4.0, 900.0, 0.0, 1.0])
    x = (sizes[:, None, None] * torch.randn(16, 3 * nkv, d, generator=g)).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    exps = []
    for t in range(16):
        ops.qk_norm_rope_write_8bit(x[t:t + 1].view(1, -1).to(dev), None, None, 1e-6, None, None, True, k, v, ks, vs,
                                    torch.tensor([16 + t], device=dev), nkv, nkv, d, err)
        exps.append((ks[1, :, 0].log2().cpu(), vs[1, :, 0].log2().cpu()))
    assert int(err.item()) == 0
    for h in range(nkv):
        for which, first in (("k", nkv), ("v", 2 * nkv)):
            true = x[:, first + h].double()
            got = (k[1, h].cpu().double() if which == "k" else v[1, h, 0].cpu().double().T)
            e = [round(float(p[0 if which == "k" else 1][h])) for p in exps]
            assert e == [exponent(true[:t + 1].abs().max().item(), dtype) for t in range(16)]
            for t in range(16):
                room = sum(half_step(true[t].abs() * 1.1, ee, dtype) for ee in sorted(set(e[t:])))
                assert ((got[t] * 2.0 ** e[-1] - true[t]).abs() <= room).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,adjacent,weight_dtype", [(128, True, torch.bfloat16), (128, False, torch.float32), (64, False, torch.bfloat16)])
def test_write_keys_have_the_codes_of_the_formula_in_64_bits(dtype, d, adjacent, weight_dtype):
    """160 x 4 keys of d elements, rounded to 32 bits, to bfloat16 and to their codes: none may differ.  (What the kernel drops
    before the first of these roundings is below 2^-40 of a value, so the chance that one differs is below 1e-6.)"""
    dev, ops = need_gpu(), _ops()
    T, nkv, page = 160, 4, 32
    g = torch.Generator().manual_seed(d + adjacent)
    qkv = torch.randn(T, 2 * nkv, d, generator=g).to(torch.bfloat16)
    kw = (1 + 0.3 * torch.randn(d, generator=g)).to(weight_dtype)
    angle = 100 * torch.rand(T, d // 2, generator=g).double()
    cos, sin = angle.cos().float(), angle.sin().float()
    k, v, ks, vs = ops.cache_8bit_pools(T // page, nkv, page, d, dtype, dev)
    ops.qk_norm_rope_write_8bit(qkv.view(T, -1).to(dev), kw.to(dev), kw.to(dev), 1e-6, cos.to(dev), sin.to(dev), adjacent, k, v, ks, vs,
                                torch.arange(T, device=dev), 0, nkv, d, torch.zeros(1, dtype=torch.int32, device=dev))
    x = qkv[:, :nkv].double()
    x = x / (x.square().mean(-1, keepdim=True) + torch.tensor(1e-6).double()).sqrt() * kw.double()
    one, two = (slice(0, d, 2), slice(1, d, 2)) if adjacent else (slice(0, d // 2), slice(d // 2, d))
    c, s = cos.double()[:, None], sin.double()[:, None]
    want = torch.empty_like(x)
    want[..., one], want[..., two] = x[..., one] * c - x[..., two] * s, x[..., one] * s + x[..., two] * c
    want = want.float().to(torch.bfloat16).double()
    got = ops.pages_8bit_to_bf16(k, v, ks, vs, torch.arange(T // page, dtype=torch.int32, device=dev))[0].cpu().double().transpose(1, 2).reshape(T, nkv, d)
    for b in range(0, T, 16):
        for h in range(nkv):
            e = exponent(want[b:b + 16, h].abs().max().item(), dtype)
            assert torch.equal(got[b:b + 16, h], encode(want[b:b + 16, h] * 2.0 ** -e, dtype) * 2.0 ** e), (b, h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm,rot", [(False, False), (False, True), (True, True)])
def test_write_keys_that_are_no_numbers(dtype, norm, rot):
    """Not-a-number keys become zeros and infinite ones the largest number of their block's scale; rows beside them are not
    touched by it (but share the scale).  A row with an infinity has no norm: all of it becomes zero."""
    dev, ops = need_gpu(), _ops()
    d, T = 64, 16
    qkv = torch.randn(T, 2, d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    qkv[2, 0, 7] = float("nan")
    qkv[3, 0, 8] = -float("inf")
    qkv[4, 0] = 0
    w = torch.ones(d, dtype=torch.bfloat16, device=dev) if norm else None
    turn = torch.full((T, d // 2), 0.6, device=dev), torch.full((T, d // 2), 0.8, device=dev)
    k, v, ks, vs = ops.cache_8bit_pools(1, 1, 16, d, dtype, dev)
    ops.qk_norm_rope_write_8bit(qkv.view(T, -1).to(dev), w, w, 1e-6, turn[0] if rot else None, turn[1] if rot else None, True, k, v, ks, vs,
                                torch.arange(T, device=dev), 0, 1, d, torch.zeros(1, dtype=torch.int32, device=dev))
    top = 448.0 if dtype == torch.float8_e4m3fn else 127.0
    got = (ops.pages_8bit_to_bf16(k, v, ks, vs, torch.zeros(1, dtype=torch.int32, device=dev))[0][0, 0].double() / ks.double().view(())).cpu()
    assert torch.isfinite(got).all() and (got[4] == 0).all()
    if norm:                                          # the sum of squares is no number, or infinite
        assert (got[2] == 0).all() and (got[3, [i for i in range(d) if i not in (8, 9)]] == 0).all()
        return
    assert ks.item() == 2.0 ** 40
    assert got[2, 7] == 0 and (got[2, 6] == 0 or not rot)
    assert got[3, 8] == -top and (got[3, 9] == -top if rot else abs(got[3, 9]) < 1)


def test_write_counts_slots_outside_the_pool():
    dev, ops = need_gpu(), _ops()
    pools = ops.cache_8bit_pools(3, 2, 16, 64, torch.int8, dev)
    qkv = torch.randn(4, 6 * 64, device=dev).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    slots = torch.tensor([-1, 48, 16, 2 ** 40], device=dev)
    q = ops.qk_norm_rope_write_8bit(qkv, None, None, 1e-6, None, None, True, *pools, slots, 2, 2, 64, err)
    assert int(err.item()) == 3 * 4 and torch.equal(q, qkv[:, :128])
    assert not pools[0].view(torch.uint8)[[0, 2]].any() and pools[0].view(torch.uint8)[1].any()


# ---- reading back ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nkv,d,page", [(2, 64, 16), (1, 128, 64), (3, 128, 16), (2, 64, 128)])
def test_pages_to_bf16_are_exact(dtype, nkv, d, page):
    dev, ops = need_gpu(), _ops()
    pools = Pools(5, nkv, page, d, dtype, seed=3)
    g = torch.Generator().manual_seed(1)
    for p in (0, 2, 4):
        pools.put(p, 0, torch.randn(page, nkv, d, generator=g).double() * 10.0 ** (p - 2), torch.randn(page, nkv, d, generator=g).double())
    ids = torch.tensor([4, -1, 0, 2, 2, 5, 1000000], dtype=torch.int32)
    spans = torch.tensor([[0, page], [0, page], [3, page - 5], [0, 0], [7, 9], [0, page], [0, page]], dtype=torch.int32)
    for use in (False, True):
        keys, values = ops.pages_8bit_to_bf16(*pools.on(dev), ids.to(dev), spans.to(dev) if use else None)
        for i, p in enumerate(ids.tolist()):
            k = torch.zeros(nkv, page, d, dtype=torch.float64); v = torch.zeros_like(k)
            if 0 <= p < 5:
                lo, hi = spans[i].tolist() if use else (0, page)
                if hi > lo:
                    a, b = pools.values(p, lo, hi - lo)
                    k[:, lo:hi], v[:, lo:hi] = a.transpose(0, 1), b.transpose(0, 1)
            assert torch.equal(keys[i].cpu().double(), k) and torch.equal(values[i].cpu().double(), v)
    # into buffers that are larger: what lies behind stays
    big = [torch.full((9, nkv, page, d), 7.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    ops.pages_8bit_to_bf16(*pools.on(dev), ids.to(dev), None, keys=big[0], values=big[1])
    assert (big[0][7:] == 7).all() and (big[1][7:] == 7).all() and torch.equal(big[0][0], keys[0])


# ---- decode attention ----------------------------------------------------------------------------------------------------
def _decode(ops, dev, dtype, lengths, nq, nkv, d, page, window=None, seed=0, value_scale=None, workspace=None, span_min=None,
            pair_cost=None, q_scale=1.0, bad_row=None):
    seqs = Sequences(lengths, nkv, d, page, dtype, seed, value_scale)
    g = torch.Generator().manual_seed(seed + 77)
    order = torch.randperm(len(lengths), generator=g).tolist()
    meta = segments_to_device([(s, lengths[s] - 1, 1) for s in order], dev)
    wide = nq * d + 24
    q = (q_scale * torch.randn(len(lengths), wide, generator=g)).to(torch.bfloat16)
    scale = 1.0 / math.sqrt(d)
    out = ops.attention_decode_8bit(q.to(dev), wide, *seqs.pools.on(dev), seqs.table.to(dev), meta["seg_off"], meta["seg_slot"],
                                    meta["seg_start"], meta["seg_len"], len(lengths), len(lengths), nq, nkv, d, window, scale,
                                    workspace=workspace, span_min=span_min, pair_cost=pair_cost)
    got = out.cpu().double().view(-1, nq, d)
    for i, s in enumerate(order):
        want, bound = attention_with_bound(q[i, :nq * d].double().view(nq, d), seqs.k[s], seqs.v[s], seqs.vs[s], lengths[s] - 1, window, scale,
                                           F16_HALF_STEP, d)
        assert ((got[i] - want).abs() <= bound).all(), (s, lengths[s], ((got[i] - want).abs() / bound).max())
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ctx", [1, 2, 15, 16, 17, 48, 63, 64, 65, 127, 128, 129, 511, 512, 513, 1300])
def test_decode_every_edge(dtype, ctx):
    _decode(_ops(), need_gpu(), dtype, [ctx], 8, 2, 128, 16, seed=ctx)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page", [(32, 8, 128, 16), (16, 1, 64, 16), (6, 3, 128, 64), (5, 5, 64, 32), (12, 1, 128, 128),
                                           (10, 2, 128, 16), (8, 1, 64, 16), (17, 1, 64, 32)])
@pytest.mark.parametrize("window", [None, 1, 100, 700])
def test_decode_many_requests(dtype, nq, nkv, d, page, window):
    _decode(_ops(), need_gpu(), dtype, [1, 700, 64, 65, 1500, 3, 130, 128], nq, nkv, d, page, window, seed=nq)


@pytest.mark.parametrize("span_min,pair_cost", [(1, 0), (3, 1), (50, 7), (5000, 0)])
@pytest.mark.parametrize("nq,nkv,d", [(8, 2, 128), (12, 1, 64)])
def test_decode_spans(span_min, pair_cost, nq, nkv, d):
    """Requests of 1 to 5,000 keys in one step, spans that cut everywhere or nowhere; a workspace full of NaN, used again."""
    dev, ops = need_gpu(), _ops()
    ws = ops.attention_decode_workspace(d, dev)
    ws.acc.fill_(float("nan")); ws.ml.fill_(float("nan"))
    for seed in range(2):
        _decode(ops, dev, torch.int8, [1, 5000, 17, 800, 64, 2000, 1, 333, 4096], nq, nkv, d, 16, None, seed, workspace=ws,
                span_min=span_min, pair_cost=pair_cost)
    assert not ws.count.any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_blocks_of_very_unequal_scales(dtype):
    """Values whose blocks differ by 2^30, the largest where no weight is: nothing is lost next to them."""
    _decode(_ops(), need_gpu(), dtype, [900, 70], 4, 2, 128, 16, seed=3, value_scale=lambda t: torch.exp2(((t // 16) % 7) * 5 - 15))
    _decode(_ops(), need_gpu(), dtype, [300], 4, 2, 64, 16, seed=4, value_scale=lambda t: torch.where(t < 100, 0.0, 1.0), q_scale=6.0)


def test_decode_large_and_small_queries():
    for q_scale in (1e-4, 30.0):
        _decode(_ops(), need_gpu(), torch.float8_e4m3fn, [200, 65], 8, 2, 128, 16, seed=8, q_scale=q_scale)


def test_decode_missing_pages_and_slots():
    """Pages that are not there are passed over; a request without any gets zeros; nothing is read out of bounds."""
    dev, ops = need_gpu(), _ops()
    seqs = Sequences([100, 40, 20], 2, 64, 16, torch.int8)
    table = seqs.table.clone()
    table[0, 2] = -1; table[0, 3] = 10 ** 6
    table[1, :] = -1
    meta = segments_to_device([(0, 99, 1), (1, 39, 1), (50, 19, 1), (2, 10 ** 6, 1), (2, 5, 3)], dev)
    q = torch.randn(7, 4 * 64, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    out = torch.full((7, 256), 9.0, dtype=torch.bfloat16, device=dev)
    ops.attention_decode_8bit(q.to(dev), 256, *seqs.pools.on(dev), table.to(dev), meta["seg_off"], meta["seg_slot"], meta["seg_start"],
                              meta["seg_len"], 7, 5, 4, 2, 64, None, 0.125, out=out)
    got = out.cpu().double()
    keep = [i for i in range(100) if not 32 <= i < 64]
    want, bound = attention_with_bound(q[0].double().view(4, 64), seqs.k[0][keep], seqs.v[0][keep], seqs.vs[0][keep], len(keep) - 1, None, 0.125, F16_HALF_STEP, 64)
    assert ((got[0].view(4, 64) - want).abs() <= bound).all()
    assert (got[1:3] == 0).all() and torch.isfinite(got[3]).all() and (got[4:] == 9).all()


@pytest.mark.parametrize("window", [None, 20])
def test_decode_padded_with_segments_of_no_length(window):
    """Segments without tokens in front, between and behind; their slots, starts and offsets may be anything."""
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page, lengths = 8, 2, 64, 16, [130, 1, 47]
    seqs = Sequences(lengths, nkv, d, page, torch.int8, 3)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.randn(5, nq * d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = torch.full((5, nq * d), 3.0, dtype=torch.bfloat16, device=dev)
    pools, table = seqs.pools.on(dev), seqs.table.to(dev)
    ops.attention_decode_8bit(q.to(dev), nq * d, *pools, table, i32(0, 0, 1, 1, 2, 3, -9), i32(99, 0, -1, 1, 2, 2 ** 31 - 1, 0),
                              i32(7, lengths[0] - 1, -5, lengths[1] - 1, lengths[2] - 1, 2 ** 31 - 1, 0), i32(0, 1, 0, 1, 1, 0, 0), 5, 7, nq, nkv, d,
                              window, 0.125, out=out)
    got = out.cpu().double().view(5, nq, d)
    for i, n in enumerate(lengths):
        want, bound = attention_with_bound(q[i].double().view(nq, d), seqs.k[i], seqs.v[i], seqs.vs[i], n - 1, window, 0.125, F16_HALF_STEP, d)
        assert ((got[i] - want).abs() <= bound).all()
    assert (got[3:] == 3).all()
    ops.attention_decode_8bit(q.to(dev), nq * d, *pools, table, i32(0), i32(0), i32(9), i32(0), 5, 1, nq, nkv, d, window, 0.125, out=out)
    assert torch.equal(out.cpu().double().view(5, nq, d), got)                  # nothing to do at all


def test_decode_is_the_same_in_a_graph_and_on_another_stream():
    dev, ops = need_gpu(), _ops()
    seqs = Sequences([700, 65, 2000], 2, 128, 16, torch.float8_e4m3fn)
    meta = segments_to_device([(i, n - 1, 1) for i, n in enumerate([700, 65, 2000])], dev)
    q = torch.randn(3, 8 * 128, device=dev).to(torch.bfloat16)
    pools, table = seqs.pools.on(dev), seqs.table.to(dev)
    ws = ops.attention_decode_workspace(128, dev)
    call = lambda: ops.attention_decode_8bit(q, 1024, *pools, table, meta["seg_off"], meta["seg_slot"], meta["seg_start"],  # noqa: E731
                                             meta["seg_len"], 3, 3, 8, 2, 128, None, 0.1, workspace=ws)
    want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for _ in range(3):
        got.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    meta["seg_start"][2] = 1000                        # a replayed step takes its lengths from the device
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, call()) and not torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    side.synchronize()
    assert torch.equal(again, got)


def test_decode_far_into_a_large_pool():
    """Pages whose bytes begin beyond 2^32."""
    dev, ops = need_gpu(), _ops()
    nkv, d = 8, 128
    pages = (1 << 32) // (nkv * 16 * d) + 40
    k, v, ks, vs = ops.cache_8bit_pools(pages, nkv, 16, d, torch.int8, dev)
    g = torch.Generator(device=dev).manual_seed(0)
    T = 40
    qkv = torch.randn(T, 3 * nkv * d, device=dev, generator=g).to(torch.bfloat16)
    ids = torch.tensor([pages - 1, pages - 30, 5], device=dev)
    slots = ids[torch.arange(T, device=dev) // 16] * 16 + torch.arange(T, device=dev) % 16
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    q = ops.qk_norm_rope_write_8bit(qkv, None, None, 1e-6, None, None, True, k, v, ks, vs, slots, nkv, nkv, d, err)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = ids.int().view(1, 3)
    out = ops.attention_decode_8bit(q[T - 1:], nkv * d, k, v, ks, vs, table, i32([0]), i32([0]), i32([T - 1]), i32([1]), 1, 1, nkv, nkv, d,
                                    None, 0.1)
    keys, values = ops.pages_8bit_to_bf16(k, v, ks, vs, table.view(-1))
    kk = keys.double().cpu().permute(0, 2, 1, 3).reshape(48, nkv, d)[:T]
    vv = values.double().cpu().permute(0, 2, 1, 3).reshape(48, nkv, d)[:T]
    x = qkv.double().cpu().view(T, 3 * nkv, d)
    assert ((kk - x[:, nkv:2 * nkv]).abs() <= 2.0 ** -6 * x[:, nkv:2 * nkv].abs().max()).all()      # half a step of 1/64 of the range
    sc = vs[ids].double().cpu().permute(0, 2, 1).repeat_interleave(16, 1).reshape(48, nkv)[:T]
    want, bound = attention_with_bound(q[T - 1].double().cpu().view(nkv, d), kk, vv, sc, T - 1, None, 0.1, F16_HALF_STEP, d)
    assert ((out.cpu().double().view(nkv, d) - want).abs() <= bound).all()


# ---- a step: maps, write, prompt and decode attention together -----------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page,window", [(8, 2, 128, 16, None), (6, 6, 64, 32, 70), (10, 2, 128, 64, 333), (4, 1, 64, 128, None)])
def test_a_step_of_portions_and_single_tokens(dtype, nq, nkv, d, page, window):
    dev, ops = need_gpu(), _ops()
    segs = [(3, 0, 200), (0, 37, 1), (5, 150, 2), (1, 0, 1), (2, 600, 129), (4, 301, 1)]     # (slot, start, length)
    g = torch.Generator().manual_seed(nq + page)
    T = sum(n for _, _, n in segs)
    per = [(a + n + page - 1) // page for _, a, n in segs]
    total = sum(per) + 3
    perm = torch.randperm(total, generator=g).tolist()
    table = torch.full((7, max(per) + 1), -1, dtype=torch.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    slot_, start, length = i32([s for s, _, _ in segs]), i32([a for _, a, _ in segs]), i32([n for _, _, n in segs])
    for (s, _, _), n in zip(segs, per):
        table[s, :n] = torch.tensor([perm.pop() for _ in range(n)], dtype=torch.int32)
    table_dev = table.to(dev)
    pools = Pools(total, nkv, page, d, dtype, seed=2).on(dev)                # random bytes, NaN scales
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    width = (nq + 2 * nkv) * d
    # what the requests hold before the step, written by an earlier one
    old = [(s, 0, a) for s, a, _ in segs if a > 0]
    m0 = ops.page_maps(table_dev, i32([s for s, _, _ in old]), i32([0] * len(old)), i32([a for _, _, a in old]), page, sum(a for _, _, a in old))
    ops.qk_norm_rope_write_8bit(torch.randn(m0.positions.numel(), width, device=dev).to(torch.bfloat16), None, None, 1e-6, None, None,
                                True, *pools, m0.slot_map, nq, nkv, d, err)
    listed = sum((a + n - 1) // page - (max(0, a - window + 1) // page if window else 0) + 1 for _, a, n in segs if n > 1)
    maps = ops.page_maps(table_dev, slot_, start, length, page, T, num_listed_pages=listed, window=window, min_tokens=2)
    qkv = torch.randn(T, width, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).to(torch.bfloat16)
    q = ops.qk_norm_rope_write_8bit(qkv, None, None, 1e-6, None, None, True, *pools, maps.slot_map, nq, nkv, d, err)
    scale = 1.0 / math.sqrt(d)
    out = torch.full((T, nq * d), 9.0, dtype=torch.bfloat16, device=dev)
    ops.attention_prompt_8bit(q, nq * d, *pools, maps, start, length, [(a, n) for _, a, n in segs if n > 1], T, nq, nkv, d, window, scale, out=out)
    singles = [int(maps.seg_off[i]) for i, (_, _, n) in enumerate(segs) if n == 1]
    assert (out[singles] == 9).all()                                          # left to the decode kernel
    ops.attention_decode_8bit(q, nq * d, *pools, table_dev, maps.seg_off, slot_, start, length, T, len(segs), nq, nkv, d, window, scale, out=out)
    assert int(err.item()) == 0 and ops.attention_tcgen05_loaded_status() == 0
    got, qd = out.cpu().double().view(T, nq, d), q.cpu().double().view(T, nq, d)
    t = 0
    for s, a, n in segs:
        ids = table[s, :(a + n + page - 1) // page].to(dev)
        k, v = (x.cpu().double().permute(0, 2, 1, 3).reshape(-1, nkv, d) for x in ops.pages_8bit_to_bf16(*pools, ids))
        sc = pools[3][ids.long()].double().cpu().permute(0, 2, 1).repeat_interleave(16, 1).reshape(-1, nkv)
        for i in range(n):
            if n == 1 or i in (0, 1, n // 2, n - 1):
                # the prompt kernel rounds its weights to bfloat16, which may reach its sum as well
                rounding = (F16_HALF_STEP, 0.0) if n == 1 else (BF16_HALF_STEP, BF16_HALF_STEP)
                want, bound = attention_with_bound(qd[t + i], k, v, sc, a + i, window, scale, rounding[0], d, rounding[1])
                assert ((got[t + i] - want).abs() <= bound).all(), (s, i, ((got[t + i] - want).abs() / bound).max())
        t += n


def test_a_step_recorded_and_replayed():
    """Maps, page write, prompt (with shares of the keys) and decode attention in one CUDA graph: replayed over pages put back to
    what they were, and again with other lengths and inputs in the same tensors, they give what the launched kernels give."""
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page, T = 8, 2, 128, 16, 60
    segs = [(0, 3000, 40), (2, 77, 1), (1, 0, 18), (3, 500, 1)]
    other = [(0, 2990, 38), (2, 79, 1), (1, 5, 18), (3, 498, 1)]                # what a replay meets; two rows are not used
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.randperm(4 * 200, generator=torch.Generator().manual_seed(6)).int().view(4, 200).to(dev)
    old = Pools(4 * 200, nkv, page, d, torch.int8, seed=5).on(dev)
    old[2].fill_(2.0 ** -5); old[3].fill_(2.0 ** -6)
    pools = [x.clone() for x in old]
    slot, start, length = (i32([s[k] for s in segs]) for k in range(3))
    qkv = torch.randn(T, (nq + 2 * nkv) * d, device=dev).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = ops.attention_decode_workspace(d, dev)
    out = torch.zeros(T, nq * d, dtype=torch.bfloat16, device=dev)

    def step():
        out.zero_()
        maps = ops.page_maps(table, slot, start, length, page, T, num_listed_pages=200, min_tokens=2)
        q = ops.qk_norm_rope_write_8bit(qkv, None, None, 1e-6, None, None, True, *pools, maps.slot_map, nq, nkv, d, err)
        ops.attention_prompt_8bit(q, nq * d, *pools, maps, start, length, [(3000, 40), (0, 18)], T, nq, nkv, d, None, d ** -0.5, out=out)
        ops.attention_decode_8bit(q, nq * d, *pools, table, maps.seg_off, slot, start, length, T, 4, nq, nkv, d, None, d ** -0.5,
                                  workspace=ws, out=out)

    def back():
        for x, y in zip(pools, old):
            x.view(torch.uint8).copy_(y.view(torch.uint8))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for now in (segs, other):
        start.copy_(i32([s[1] for s in now])); length.copy_(i32([s[2] for s in now]))
        qkv.copy_(torch.randn(T, (nq + 2 * nkv) * d, device=dev))
        results = []
        for run in (step, graph.replay, graph.replay):
            back()
            run()
            torch.cuda.synchronize()
            results.append([out.clone()] + [x.view(torch.uint8).clone() for x in pools])
        used = sum(s[2] for s in now)
        assert not (results[0][0][:used] == 0).all(1).any() and (results[0][0][used:] == 0).all()
        for again in results[1:]:
            assert all(torch.equal(x, y) for x, y in zip(results[0], again))
    # the slot map is -1 behind the last token: two rows, counted once per key and value head in three of the calls
    assert int(err.item()) == 3 * 2 * 2 * nkv and ops.attention_tcgen05_loaded_status() == 0


@pytest.mark.parametrize("fit", [1, 90, 200, 333])
@pytest.mark.parametrize("start", [0, 5000])
def test_portions_with_more_tokens_than_rows(fit, start):
    # the maps, the queries and the output hold the first `fit` of 200 + 150 tokens: the others are left out, and nothing is
    # written behind the last row (start 5000: with shares of the keys)
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page = 8, 2, 64, 16
    portions = [(start, 200), (0, 150)]
    g = torch.Generator().manual_seed(fit)
    per = [(a + n + page - 1) // page for a, n in portions]
    table = torch.full((2, max(per)), -1, dtype=torch.int32)
    perm = torch.randperm(sum(per), generator=g).int()
    table[0, :per[0]], table[1, :per[1]] = perm[:per[0]], perm[per[0]:]
    pools = tuple(x.to(dev) for x in ops.cache_8bit_pools(sum(per), nkv, page, d, torch.int8, "cpu"))
    pools[0].view(torch.uint8).random_(0, 256)
    pools[1].view(torch.uint8).random_(0, 256)
    for x in pools[2:]:
        x.fill_(2.0 ** -6)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    s_, l_ = i32([a for a, _ in portions]), i32([n for _, n in portions])
    q = torch.randn(350, nq * d, device=dev).to(torch.bfloat16)
    results = []
    for tokens in (350, fit):
        maps = ops.page_maps(table.to(dev), i32([0, 1]), s_, l_, page, tokens, num_listed_pages=sum(per), min_tokens=2)
        buffer = torch.full((352, nq * d), 7.0, dtype=torch.bfloat16, device=dev)
        ops.attention_prompt_8bit(q[:tokens], nq * d, *pools, maps, s_, l_, portions, tokens, nq, nkv, d, None, d ** -0.5, out=buffer[:tokens])
        assert ops.attention_tcgen05_loaded_status() == 0 and (buffer[tokens:] == 7).all()
        results.append(buffer[:fit].double())
    assert not (results[1] == 7).all(1).any()
    # the shares of the keys may be cut elsewhere: weights and output round to bfloat16, twice each
    bound = 4 * 2.0 ** -8 * pools[1].view(torch.int8).abs().max().item() * 2.0 ** -6
    assert (results[0] - results[1]).abs().max().item() <= bound


# ---- refusals ---------------------------------------------------------------------------------------------------------
def _refused(call, *words):
    from pulse_infer_b200.ops import KernelError
    with pytest.raises(KernelError) as info:
        call()
    for w in words:
        assert w in str(info.value), str(info.value)


def test_what_the_cache_kernels_refuse():
    dev, ops = need_gpu(), _ops()
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=dev)  # noqa: E731
    bf = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=dev)  # noqa: E731
    f32 = lambda *shape: torch.zeros(shape, device=dev)  # noqa: E731
    k, v, ks, vs = pools = ops.cache_8bit_pools(2, 2, 16, 64, torch.int8, dev)
    for bad in ((1, 2, 8, 64, torch.int8), (1, 2, 48, 64, torch.int8), (1, 2, 16, 96, torch.int8), (1, 2, 16, 64, torch.uint8)):
        _refused(lambda: ops.cache_8bit_pools(*bad, dev), "no 8-bit pages")
    # page maps
    maps = lambda **kw: ops.page_maps(**{**dict(block_table=i32(2, 3), seg_slot=i32(2), seg_start=i32(2), seg_len=i32(2), page_size=16,  # noqa: E731
                                                num_tokens=2), **kw})
    maps()
    for kw in (dict(page_size=24), dict(page_size=0), dict(num_tokens=-1), dict(num_listed_pages=-1), dict(window=0), dict(min_tokens=0),
               dict(seg_len=i32(3)), dict(seg_start=i32(2).long()), dict(block_table=i32(6)), dict(block_table=i32(3, 2).T),
               dict(seg_slot=i32(0), seg_start=i32(0), seg_len=i32(0)), dict(seg_slot=i32(4097), seg_start=i32(4097), seg_len=i32(4097))):
        _refused(lambda: maps(**kw))
    # the write
    T, nq, nkv, d = 3, 4, 2, 64
    base = dict(qkv=bf(T, (nq + 2 * nkv) * d), q_weight=bf(d), k_weight=bf(d), eps=1e-6, cos=f32(T, 32), sin=f32(T, 32), adjacent_pairs=True,
                kcache=k, vcache=v, kscale=ks, vscale=vs, slot_map=torch.arange(T, device=dev), nq=nq, nkv=nkv, head_dim=d, error_count=i32(1))
    ops.qk_norm_rope_write_8bit(**base)
    for kw in (dict(qkv=bf(T, 8 * d).float()), dict(qkv=bf(T, 9 * d)), dict(qkv=bf(8 * d, T).T), dict(q_weight=bf(d + 1)), dict(k_weight=None),
               dict(k_weight=f32(d)), dict(cos=None), dict(cos=f32(T, 33), sin=f32(T, 33)), dict(cos=f32(T, 6), sin=f32(T, 6)),
               dict(cos=f32(T, 12), sin=f32(T, 12), adjacent_pairs=False), dict(slot_map=i32(T)), dict(slot_map=torch.arange(T + 1, device=dev)),
               dict(error_count=f32(1)), dict(vcache=v.view(2, 2, 16, 64)), dict(kscale=f32(2, 2)), dict(vscale=vs.double()), dict(nkv=1, nq=6),
               dict(head_dim=128), dict(kcache=k.to(torch.float16)), dict(kcache=k.float().to(torch.float8_e4m3fn)), dict(q_out=bf(T, 3)),
               dict(kcache=torch.empty(2, 2, 64, 16, dtype=torch.int8, device=dev).transpose(2, 3))):
        _refused(lambda: ops.qk_norm_rope_write_8bit(**{**base, **kw}))
    # reading back
    _refused(lambda: ops.pages_8bit_to_bf16(*pools, torch.zeros(2, dtype=torch.int64, device=dev)))
    _refused(lambda: ops.pages_8bit_to_bf16(*pools, i32(2), i32(2)))
    _refused(lambda: ops.pages_8bit_to_bf16(*pools, i32(2), keys=bf(1, 2, 16, 64)))
    a, b = ops.pages_8bit_to_bf16(*pools, i32(0))
    assert a.shape == (0, 2, 16, 64)
    # attention
    base = dict(q=bf(2, nq * d), q_stride=nq * d, kcache=k, vcache=v, kscale=ks, vscale=vs, block_table=i32(2, 2), seg_off=torch.tensor([0, 1], dtype=torch.int32, device=dev),
                seg_slot=i32(2), seg_start=i32(2), seg_len=i32(2) + 1, num_tokens=2, num_segments=2, nq=nq, nkv=nkv, head_dim=d, window=None, scale=0.1)
    ops.attention_decode_8bit(**base)
    for kw in (dict(q=bf(2, nq * d).float()), dict(q_stride=nq * d - 8), dict(q_stride=nq * d + 8), dict(q_stride=nq * d + 4), dict(nq=3), dict(scale=0.0),
               dict(scale=float("nan")), dict(window=0), dict(window=-5), dict(num_segments=3), dict(seg_len=i32(2).float()), dict(block_table=i32(4)),
               dict(out=bf(2, 8)), dict(out=f32(2, nq * d)), dict(span_min=0), dict(pair_cost=65), dict(head_dim=128), dict(num_tokens=3),
               dict(workspace=ops.attention_decode_workspace(32, dev)),
               dict(num_segments=1025, seg_off=i32(1025), seg_slot=i32(1025), seg_start=i32(1025), seg_len=i32(1025))):
        _refused(lambda: ops.attention_decode_8bit(**{**base, **kw}))
    got = maps(num_listed_pages=1)
    base = dict(q=bf(2, nq * d), q_stride=nq * d, kcache=k, vcache=v, kscale=ks, vscale=vs, maps=got, seg_start=i32(2), seg_len=i32(2), portions=[(0, 2)],
                num_tokens=2, nq=nq, nkv=nkv, head_dim=d, window=None, scale=0.1)
    for kw in (dict(portions=[(15, 2)]), dict(q=bf(2, nq * d).float()), dict(seg_len=i32(1)), dict(window=0), dict(out=bf(1, 1))):
        _refused(lambda: ops.attention_prompt_8bit(**{**base, **kw}))


def test_outputs_off_their_boundaries_are_refused():
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page = 2, 1, 64, 16
    pools = ops.cache_8bit_pools(4, nkv, page, d, torch.int8, dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table, start, length = i32(0, 1).view(1, 2), i32(0), i32(3)
    maps = ops.page_maps(table, i32(0), start, length, page, 3, num_listed_pages=1, min_tokens=2)
    buffer = torch.zeros(4 * nq * d, dtype=torch.bfloat16, device=dev)
    q = torch.randn(3, nq * d, device=dev).to(torch.bfloat16)
    for off, prompt, decode in ((0, True, True), (8, True, True), (4, False, True), (1, False, False), (2, False, False)):
        out = buffer[off:off + 3 * nq * d].view(3, nq * d)
        call = lambda: ops.attention_prompt_8bit(q, nq * d, *pools, maps, start, length, [(0, 3)], 3, nq, nkv, d, None, 0.1, out=out)  # noqa: E731
        call() if prompt else _refused(call, "16-byte")
        one = buffer[off:off + nq * d].view(1, nq * d)
        call = lambda: ops.attention_decode_8bit(q[:1], nq * d, *pools, table, maps.seg_off, i32(0), start, i32(1), 1, 1, nq, nkv, d, None,  # noqa: E731
                                                 0.1, out=one)
        call() if decode else _refused(call, "8-byte")
    torch.cuda.synchronize()
    keys = torch.zeros(8 + nkv * page * d, dtype=torch.bfloat16, device=dev)
    _refused(lambda: ops.pages_8bit_to_bf16(*pools, i32(0), keys=keys[1:1 + nkv * page * d].view(1, nkv, page, d)), "16-byte")
    _refused(lambda: ops.attention_prompt_8bit(q, nq * d, *pools, maps, start, length, [(30, 3)], 3, nq, nkv, d, None, 0.1), "beyond a block table")


@pytest.mark.parametrize("requests", [257, 1024])
def test_decode_a_great_many_short_requests(requests):
    """More requests than threads in a block, most of them a tile or two long, some of no length at all."""
    lengths = [1 + (i * 37) % 70 for i in range(requests)]
    lengths[5] = 900
    _decode(_ops(), need_gpu(), torch.int8, lengths, 2, 1, 64, 16, seed=requests)


def test_calls_without_tokens():
    dev, ops = need_gpu(), _ops()
    pools = ops.cache_8bit_pools(2, 2, 16, 64, torch.float8_e4m3fn, dev)
    before = [p.clone() for p in pools]
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    q = ops.qk_norm_rope_write_8bit(torch.empty(0, 512, dtype=torch.bfloat16, device=dev), None, None, 1e-6, None, None, True, *pools,
                                    torch.empty(0, dtype=torch.int64, device=dev), 4, 2, 64, err)
    assert q.shape == (0, 256) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(pools, before))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.zeros(3, 256, dtype=torch.bfloat16, device=dev)
    out = torch.full((3, 256), 5.0, dtype=torch.bfloat16, device=dev)
    for start, length in (((0, 3), (0, 3)), ((-4, 0), (1, 0))):           # no segment of one token, or one at no position
        ops.attention_decode_8bit(q, 256, *pools, torch.zeros(2, 2, dtype=torch.int32, device=dev), i32(0, 0), i32(0, 1), i32(*start),
                                  i32(*length), 3, 2, 4, 2, 64, None, 0.1, out=out)
        assert (out == 5).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nq,nkv,d,page,window", [(8, 2, 128, 16, None), (4, 4, 64, 64, None), (6, 2, 64, 16, 90), (4, 1, 128, 128, None)])
def test_portions_over_missing_pages(dtype, nq, nkv, d, page, window):
    """Pages that are not in the block table, or not in the pool, are left out of the softmax, as single tokens leave them out: in
    the middle of a context, at its beginning, under the portion itself; with shares of the keys and without; all of them."""
    dev, ops = need_gpu(), _ops()
    for portions in ([(300, 40), (0, 200), (257, 3), (64, 70)], [(3000, 20), (700, 5)]):
        lengths = [a + n for a, n in portions]
        seqs = Sequences(lengths, nkv, d, page, dtype, seed=page + nq)
        table = seqs.table.clone()
        rng = np.random.RandomState(d + page)
        for s in range(len(lengths)):
            used = (lengths[s] + page - 1) // page
            for i in range(used):
                if rng.rand() < 0.3:
                    table[s, i] = [-1, 10 ** 6, seqs.pools.pages][rng.randint(3)]
        table[1, :] = -1                                   # nothing of it is there
        table[0, 0] = -1                                   # neither are the first keys of this one
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        T = sum(n for _, n in portions)
        start, length = i32([a for a, _ in portions]), i32([n for _, n in portions])
        listed = sum((a + n - 1) // page - (max(0, a - window + 1) // page if window else 0) + 1 for a, n in portions)
        maps = ops.page_maps(table.to(dev), i32(list(range(len(portions)))), start, length, page, T, num_listed_pages=listed, window=window, min_tokens=2)
        q = torch.randn(T, nq * d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        pools = seqs.pools.on(dev)
        out = ops.attention_prompt_8bit(q.to(dev), nq * d, *pools, maps, start, length, portions, T, nq, nkv, d, window, d ** -0.5)
        assert ops.attention_tcgen05_loaded_status() == 0
        got, t = out.cpu().double().view(T, nq, d), 0
        for s, (a, n) in enumerate(portions):
            there = [0 <= int(table[s, i // page]) < seqs.pools.pages for i in range(a + n)]
            for i in sorted({0, 1, n // 2, n - 2, n - 1} | set(range(0, n, 17))):
                lo = max(0, a + i - window + 1) if window else 0
                keep = [x for x in range(lo, a + i + 1) if there[x]]
                if not keep:
                    assert (got[t + i] == 0).all(), (s, i)
                    continue
                want, bound = attention_with_bound(q[t + i].double().view(nq, d), seqs.k[s][keep], seqs.v[s][keep], seqs.vs[s][keep], len(keep) - 1,
                                                   None, d ** -0.5, BF16_HALF_STEP, d, BF16_HALF_STEP)
                assert ((got[t + i] - want).abs() <= bound).all(), (s, i, ((got[t + i] - want).abs() / bound).max())
            t += n


def test_prompt_attention_without_rows():
    """Maps and queries of no tokens at all, with portions that would be cut into shares and without: nothing to do."""
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page = 8, 2, 64, 16
    pools = ops.cache_8bit_pools(400, nkv, page, d, torch.int8, dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    for start in (0, 5000):
        table = torch.arange(400, dtype=torch.int32, device=dev).view(1, 400)
        maps = ops.page_maps(table, i32(0), i32(start), i32(30), page, 0, num_listed_pages=(start + 29) // page + 1, min_tokens=2)
        q = torch.zeros(0, nq * d, dtype=torch.bfloat16, device=dev)
        out = ops.attention_prompt_8bit(q, nq * d, *pools, maps, i32(start), i32(30), [(start, 30)], 0, nq, nkv, d, None, 0.1)
        assert out.shape == (0, nq * d)


def test_windows_beyond_32_bits():
    """A window that no context reaches is no window, however large the number."""
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page = 4, 2, 64, 16
    seqs = Sequences([200, 60], nkv, d, page, torch.int8)
    pools, table = seqs.pools.on(dev), seqs.table.to(dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.randn(11, nq * d, device=dev).to(torch.bfloat16)
    results = []
    for window in (None, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 63 - 1, 2 ** 70):
        start, length = i32(190, 59), i32(10, 1)
        maps = ops.page_maps(table, i32(0, 1), start, length, page, 11, num_listed_pages=13, window=window, min_tokens=2)
        out = torch.zeros(11, nq * d, dtype=torch.bfloat16, device=dev)
        ops.attention_prompt_8bit(q, nq * d, *pools, maps, start, length, [(190, 10)], 11, nq, nkv, d, window, 0.1, out=out)
        ops.attention_decode_8bit(q, nq * d, *pools, table, maps.seg_off, i32(0, 1), start, length, 11, 2, nq, nkv, d, window, 0.1, out=out)
        results.append((maps.page_list.clone(), maps.page_tokens.clone(), maps.table.clone(), out))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_page_maps_and_the_kernel_right_behind_them():
    """The bf16 attention kernels read offsets and slots before they wait for the kernel in front of them; here that kernel is the
    one that makes them, in memory that held the offsets of another step.  200 steps of two kinds in turn, no pause between."""
    from gpu_util import PagedKV
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page = 8, 2, 128, 16
    kinds = [[(0, 40, 30), (1, 0, 64), (2, 100, 20), (3, 7, 9)], [(3, 10, 6), (2, 60, 60), (0, 0, 41), (1, 64, 16)]]     # (slot, start, length)
    kv = PagedKV([70, 80, 120, 16], nkv, d, page, torch.bfloat16, dev)
    q = torch.randn(123, nq * d, device=dev).to(torch.bfloat16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    metas = [[i32([s[k] for s in segs]) for k in range(3)] for segs in kinds]
    # filler segments: their sums take the kernel a while
    many = 2000
    wide = [[torch.cat([x, torch.zeros(many, dtype=torch.int32, device=dev)]) for x in meta] for meta in metas]

    def step(kind, out, pause):
        slot, start, length = wide[kind]
        maps = ops.page_maps(kv.table_dev, slot, start, length, page, 123, min_tokens=2, with_table=False)
        if pause:
            torch.cuda.synchronize()
        ops.attention_tcgen05(q, nq * d, kv.kcache, kv.vcache, kv.table_dev, maps.seg_off, slot, start, length, 123, 4, 64, nq, nkv, d, page, None,
                              d ** -0.5, out)

    want, outs = ([torch.zeros(123, nq * d, dtype=torch.bfloat16, device=dev) for _ in range(n)] for n in (2, 200))
    for kind in (0, 1):
        step(kind, want[kind], True)
    torch.cuda.synchronize()
    for i in range(200):
        step(i % 2, outs[i], False)
    torch.cuda.synchronize()
    assert ops.attention_tcgen05_loaded_status() == 0 and (want[0] != 0).any() and not torch.equal(*want)
    assert all(torch.equal(out, want[i % 2]) for i, out in enumerate(outs))


def test_a_recorded_step_replayed_with_single_tokens_only():
    """The prompt kernel then finds nothing to do in any CTA; pages, queries and single tokens around it come out as launched."""
    dev, ops = need_gpu(), _ops()
    nq, nkv, d, page, T = 8, 2, 128, 16, 50
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.randperm(2 * 200, generator=torch.Generator().manual_seed(6)).int().view(2, 200).to(dev)
    old = Pools(2 * 200, nkv, page, d, torch.int8, seed=5).on(dev)
    old[2].fill_(2.0 ** -5); old[3].fill_(2.0 ** -6)
    pools = [x.clone() for x in old]
    slot, start, length = i32([0, 1]), i32([3000, 77]), i32([40, 10])
    qkv = torch.randn(T, (nq + 2 * nkv) * d, device=dev).to(torch.bfloat16)
    err = torch.zeros(1, dtype=torch.int32, device=dev)
    ws = ops.attention_decode_workspace(d, dev)
    out = torch.zeros(T, nq * d, dtype=torch.bfloat16, device=dev)

    def step():
        out.fill_(4.0)
        maps = ops.page_maps(table, slot, start, length, page, T, num_listed_pages=200, min_tokens=2)
        q = ops.qk_norm_rope_write_8bit(qkv, None, None, 1e-6, None, None, True, *pools, maps.slot_map, nq, nkv, d, err)
        ops.attention_prompt_8bit(q, nq * d, *pools, maps, start, length, [(3000, 40), (77, 10)], T, nq, nkv, d, None, d ** -0.5, out=out)
        ops.attention_decode_8bit(q, nq * d, *pools, table, maps.seg_off, slot, start, length, T, 2, nq, nkv, d, None, d ** -0.5,
                                  workspace=ws, out=out)

    def back():
        for x, y in zip(pools, old):
            x.view(torch.uint8).copy_(y.view(torch.uint8))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lengths in ([1, 1], [40, 10], [1, 1], [0, 1], [1, 0], [0, 0]):
        length.copy_(i32(lengths))
        results = []
        for run in (step, graph.replay, graph.replay):
            back()
            run()
            torch.cuda.synchronize()
            results.append([out.clone()] + [x.view(torch.uint8).clone() for x in pools])
        assert (results[0][0][sum(lengths):] == 4).all() and not (results[0][0][:sum(lengths)] == 4).all(1).any()
        for again in results[1:]:
            assert all(torch.equal(x, y) for x, y in zip(results[0], again))
    assert ops.attention_tcgen05_loaded_status() == 0
