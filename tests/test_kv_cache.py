"""The 8-bit key/value cache: quantisation into its blocks and reading back bit for bit against the definition in fp32, attention
against 64 bits.

Bound of an attention output, relative to sum p |v| of the element: a weight is rounded to fp16 once (2^-11) and its
exponent is off by at most D 2^-24 of the score's absolute products, 2^-23 of the score and 2^-21 (the exponential,
the scales' logarithms), in the numerator and in the denominator; weights below fp16's normal range are off by 2^-25 of the
largest one each; fp32 sums of `length` terms by length 2^-24; and the output is rounded once."""
import copy
import io
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import if_i_could_turn_back_time_b200 as jq
from if_i_could_turn_back_time_b200 import _lib, ops
from oracle import attention as oracle

DEV = "cuda"
gpu = pytest.mark.gpu


def _table(lengths, T, blocks, gen, width=None):
    need = [-(-n // T) for n in lengths]
    width = width or max(1, max(need))
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    free = torch.randperm(blocks, generator=gen).int()
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = free[at:at + n]
        at += n
    assert at <= blocks
    return table


def _starts(new):
    return torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)


def _filled(lengths, H, D, T, fmt, seed, spare=3, width=None):
    """A cache whose sequences hold random codes, blocks of very different scales, and what they stand for: dense [H, n, D]."""
    gen = torch.Generator().manual_seed(seed)
    blocks = sum(-(-n // T) for n in lengths) + spare
    table = _table(lengths, T, blocks, gen, width)
    cache = jq.KVCache.empty(blocks, H, D, block_size=T, fmt=fmt, device=DEV)
    dense = {}
    for what in ("keys", "values"):
        if fmt == "int8":
            codes = (torch.randn(blocks, H, T, D, generator=gen) * 40).round().clamp(-127, 127).add(128).to(torch.uint8)
        else:
            codes = (torch.randn(blocks, H, T, D, generator=gen) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        scales = torch.exp(torch.rand(blocks, H, generator=gen) * 3 - 4) / (40 if fmt == "int8" else 100) * (4 if what == "keys" else 1)
        laid = torch.empty(blocks, H, T * D, dtype=torch.uint8)
        laid[:, :, torch.from_numpy(oracle.places(T, D, what).reshape(-1))] = codes.reshape(blocks, H, T * D)
        getattr(cache, what).copy_(laid.view(blocks, H, T, D))
        getattr(cache, what[:-1] + "_scales").copy_(scales)
        real = torch.from_numpy(oracle.decode(codes.numpy(), fmt)).double() * scales.double()[..., None, None]
        dense[what] = [torch.cat([real[b] for b in row[:-(-n // T)].tolist()] or [torch.zeros(H, 0, D).double()], 1)[:, :n]
                       for row, n in zip(table, lengths)]
    return cache, table, dense


def _check_attend(q, got, lse, dense, lengths, new, window, scale=None):
    D, Hq = q.shape[-1], q.shape[1]
    scale = scale or 1 / math.sqrt(D)
    step = 2.0 ** -11 if got.dtype == torch.float16 else 2.0 ** -8
    row = 0
    for i, (n, length) in enumerate(zip(new, lengths)):
        for h in range(Hq):
            hk = h // (Hq // dense["keys"][i].shape[0])
            keys, values = dense["keys"][i][hk].to(DEV), dense["values"][i][hk].to(DEV)
            ref, want, weight, size = oracle.attend(q[row:row + n, h], keys, values, length - n, scale, window)
            err = (got[row:row + n, h].double() - ref).abs()
            off = D * 2.0 ** -24 * size + 2.0 ** -23 * size + 2.0 ** -21 + length * 2.0 ** -24
            vmax = values.abs().max() if length else torch.tensor(0.0)
            bound = (2.0 ** -11 + 2 * off)[:, None] * weight + 2.0 ** -25 * length * vmax + step * ref.abs() + (2.0 ** -24 if step < 2.0 ** -9 else 0)
            assert bool((err <= bound).all()), (i, h, (err / bound.clamp(min=1e-300)).max().item())
            if lse is not None:
                empty = torch.isinf(want)
                assert torch.equal(torch.isinf(lse[row:row + n, h]), empty)
                assert bool(((lse[row:row + n, h].double() - want).abs()[~empty] <= (off + 2.0 ** -22 * want.abs())[~empty]).all())
        row += n


ATTEND = [
    # lengths, new tokens, query heads, key heads, D, T, format, dtype, window
    ([1], [1], 1, 1, 64, 16, "int8", torch.bfloat16, 0),
    ([0, 1, 2], [1, 1, 1], 2, 2, 128, 64, "e4m3", torch.float16, 0),                      # a row that sees nothing
    ([15, 16, 17, 31, 32, 33], [1] * 6, 8, 2, 64, 16, "int8", torch.float16, 0),           # blocks of 16: half a stage
    ([63, 64, 65, 127, 128, 129], [1] * 6, 8, 1, 128, 32, "e4m3", torch.bfloat16, 0),
    ([700, 3, 0, 1111], [1, 1, 1, 1], 32, 32, 128, 64, "int8", torch.bfloat16, 0),         # one row per key head
    ([5000, 77, 2500], [1, 1, 1], 12, 4, 64, 128, "e4m3", torch.float16, 0),               # groups of three
    ([900, 1300], [1, 1], 64, 8, 128, 16, "int8", torch.bfloat16, 300),                    # a window that begins inside a stage
    ([40, 500, 9, 260], [3, 5, 1, 2], 8, 2, 64, 16, "e4m3", torch.bfloat16, 0),            # drafts
    ([33, 200], [2, 2], 8, 1, 128, 128, "int8", torch.float16, 17),                        # 16 rows
    ([70, 129, 400], [7, 0, 4], 16, 4, 128, 64, "e4m3", torch.bfloat16, 0),                # a sequence without new tokens
    ([50, 64], [50, 31], 12, 4, 64, 32, "int8", torch.bfloat16, 0),                        # prompts from the first token
    ([300], [257], 3, 1, 128, 64, "e4m3", torch.float16, 0),
    ([600, 129], [129, 128], 8, 2, 128, 64, "int8", torch.bfloat16, 100),                  # prompts with a window
    ([128, 640, 1000], [128, 1, 333], 16, 2, 64, 128, "int8", torch.float16, 0),
    ([2, 3], [5, 3], 4, 2, 64, 16, "int8", torch.bfloat16, 0),                             # more new tokens than are held: some see nothing
    ([130], [40], 128, 1, 128, 16, "e4m3", torch.bfloat16, 0),                             # a group of 128 heads
]


@gpu
@pytest.mark.parametrize("case", ATTEND, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}/{c[3]}-{c[4]}-{c[5]}-{c[6]}-w{c[8]}")
def test_attention_against_64_bits(case):
    lengths, new, Hq, H, D, T, fmt, dtype, window = case
    cache, table, dense = _filled(lengths, H, D, T, fmt, sum(lengths) + D)
    q = torch.randn(sum(new), Hq, D, generator=torch.Generator().manual_seed(5)).mul(1.5).to(dtype).to(DEV)
    args = (table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), _starts(new).to(DEV))
    got, lse = cache.attend(q, *args, max_new=max(new), window=window, lse=True)
    _check_attend(q, got, lse, dense, lengths, new, window)
    again = cache.attend(q, *args, window=window)                                          # max_new not given
    assert again.dtype == dtype and again.shape == q.shape
    assert torch.equal(cache.attend(q, *args, max_new=max(new), window=window), got)       # bit for bit
    _check_attend(q, again, None, dense, lengths, new, window)
    assert ops.check_status(raise_on_error=False) == 0


@gpu
@pytest.mark.parametrize("D,fmt", [(64, "int8"), (128, "e4m3")])
def test_one_long_sequence_over_every_sm(D, fmt):
    """Segments of more than 32 stages a warp, hundreds of parts of one pair."""
    length, T = 1250000 // (D // 64), 128
    width = -(-length // T)
    gen = torch.Generator(DEV).manual_seed(3)
    cache = jq.KVCache.empty(width, 1, D, block_size=T, fmt=fmt, device=DEV)
    for what in ("keys", "values"):
        codes = torch.randint(0, 256, cache.keys.shape, dtype=torch.uint8, device=DEV, generator=gen)
        if fmt == "e4m3":
            codes = torch.where((codes & 127) == 127, 0, codes)
        getattr(cache, what).copy_(codes)
        getattr(cache, what[:-1] + "_scales").copy_((torch.rand(width, 1, device=DEV, generator=gen) + 0.5) / 200)
    table = torch.randperm(width, device=DEV, generator=gen).int()[None].contiguous()
    lengths = torch.tensor([length], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, D, device=DEV, generator=gen).bfloat16()
    k, v = cache.read(table, lengths, length)
    dense = {"keys": [k[0].transpose(0, 1).double()], "values": [v[0].transpose(0, 1).double()]}
    got, lse = cache.attend(q, table, lengths, lse=True)
    _check_attend(q, got, lse, dense, [length], [1], 0)
    got = cache.attend(q, table, lengths, window=70001)
    _check_attend(q, got, None, dense, [length], [1], 70001)
    assert ops.check_status(raise_on_error=False) == 0


@gpu
def test_many_sequences_of_every_length():
    lengths = list(range(0, 700, 3)) + [1] * 300
    cache, table, dense = _filled(lengths, 2, 64, 32, "int8", 9)
    q = torch.randn(len(lengths), 4, 64, generator=torch.Generator().manual_seed(6)).half().to(DEV)
    got = cache.attend(q, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    _check_attend(q, got, None, dense, lengths, [1] * len(lengths), 0)


@gpu
@pytest.mark.parametrize("new", [1, 40, 200])
def test_offsets_past_32_bits(new):
    """Blocks behind the first 4 GB of the pool, a table that is a part of a wider one."""
    blocks, H, D, T = 70000, 8, 128, 64
    pool = jq.KVCache(torch.empty(blocks, H, T, D, dtype=torch.uint8, device=DEV), torch.empty(blocks, H, T, D, dtype=torch.uint8, device=DEV),
                      torch.ones(blocks, H, device=DEV), torch.ones(blocks, H, device=DEV), "int8")
    lengths = [300, 90]
    cache, table, dense = _filled(lengths, H, D, T, "int8", 4)
    shift = blocks - cache.blocks
    for name in ("keys", "values", "key_scales", "value_scales"):
        getattr(pool, name)[shift:] = getattr(cache, name)
    wide = torch.full((2, 40), 123456789, dtype=torch.int32, device=DEV)
    wide[:, 3:3 + table.shape[1]] = torch.where(table >= 0, table + shift, table).to(DEV)
    news = [new, min(new, 77)]
    q = torch.randn(sum(news), 16, D, generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    view, lens = wide[:, 3:3 + table.shape[1]], torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = pool.attend(q, view, lens, _starts(news).to(DEV), max_new=max(news))
    _check_attend(q, got, None, dense, lengths, news, 0)
    k = torch.randn(sum(news), H, D, generator=torch.Generator().manual_seed(7)).to(DEV)
    pool.append(k, k, view, lens, _starts(news).to(DEV))
    cache.append(k, k, table.to(DEV), lens, _starts(news).to(DEV))
    for a, b in zip(pool.read(view, lens, 300), cache.read(table.to(DEV), lens, 300)):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("new", [1, 3, 60, 150])
def test_strides_offsets_and_streams(new):
    """Queries, keys and values as parts of one projection; rows off a 16-byte boundary; another stream."""
    lengths, news, H, G, D = [200, 333], [new, new], 2, 4, 64
    cache, table, dense = _filled(lengths, H, D, 64, "e4m3", 11)
    table, lens = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    raw = torch.randn(2 * new * (H * G + 2 * H) * D + 1, generator=torch.Generator().manual_seed(8)).to(DEV).half()
    aligned = cache.attend(raw[:-1].view(2 * new, -1, D)[:, :H * G].contiguous(), table, lens)
    packed = raw[:-1].view(2, new, H * G + 2 * H, D)
    q = packed[:, :, :H * G]
    assert torch.equal(cache.attend(q, table, lens), aligned.view(q.shape))
    _check_attend(q.reshape(2 * new, H * G, D), aligned, None, dense, lengths, news, 0)
    off = raw[1:].view(2 * new, -1, D)[:, :H * G]
    assert torch.equal(cache.attend(off, table, lens), cache.attend(off.clone(), table, lens))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = cache.attend(q, table, lens)
    stream.synchronize()
    assert torch.equal(other, aligned.view(q.shape))
    twin = jq.KVCache(*(getattr(cache, n).clone() for n in ("keys", "values", "key_scales", "value_scales")), "e4m3")
    k, v = packed[:, :, H * G:H * G + H], packed[:, :, H * G + H:]
    cache.append(k, v, table, lens)
    twin.append(k.reshape(-1, H, D).clone(), v.reshape(-1, H, D).clone(), table, lens)
    off = raw[1:].view(2 * new, -1, D)
    for x in (cache, twin):
        x.append(*((off[:, :H], off[:, H:2 * H]) if x is cache else (off[:, :H].clone(), off[:, H:2 * H].clone())), table, lens)
    assert torch.equal(cache.keys, twin.keys) and torch.equal(cache.values, twin.values)
    assert torch.equal(cache.key_scales, twin.key_scales) and torch.equal(cache.value_scales, twin.value_scales)


@gpu
@pytest.mark.parametrize("new,G", [(1, 1), (1, 8), (5, 4), (64, 2), (300, 1)])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_what_lies_outside_a_sequence_does_not_matter(new, G, fmt):
    """Every code behind the ends, every block that no sequence owns and every table entry behind the last one is the worst
    there is (NaN codes, infinite scales, ids that name nothing); entries that name nothing inside a sequence hide their tokens."""
    lengths, H, D, T = [301, 450], 2, 64, 32
    cache, table, dense = _filled(lengths, H, D, T, fmt, 13, spare=5, width=20)
    used = torch.zeros(cache.blocks, dtype=torch.bool)
    for row, n in zip(table, lengths):
        used[row[:-(-n // T)].long()] = True
    bad = 0x7F if fmt == "e4m3" else 0xFF
    for what in ("keys", "values"):
        codes = getattr(cache, what)
        codes[~used.to(DEV)] = bad
        getattr(cache, what[:-1] + "_scales")[~used.to(DEV)] = math.inf
        place = torch.from_numpy(oracle.places(T, D, what))
        for row, n in zip(table, lengths):
            if n % T:
                last = codes[int(row[n // T])].view(H, T * D)
                last[:, place[n % T:].reshape(-1).to(DEV)] = bad
    table = torch.where(table < 0, torch.tensor(2 ** 31 - 1, dtype=torch.int32), table)
    q = torch.randn(2 * new, H * G, D, generator=torch.Generator().manual_seed(9)).bfloat16().to(DEV)
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = cache.attend(q, table.to(DEV), lens)
    _check_attend(q, got, None, dense, lengths, [new] * 2, 0)
    hidden = table.clone()
    hidden[0, 2], hidden[1, 0], hidden[1, 14] = -1, cache.blocks, -2 ** 31
    got = cache.attend(q, hidden.to(DEV), lens)
    assert torch.isfinite(got).all()
    gone = {0: [2], 1: [0, 14]}
    row = 0
    for i, length in enumerate(lengths):
        keep = torch.tensor([t // T not in gone[i] for t in range(length)])
        for h in range(H * G):
            keys, values = dense["keys"][i][h // G].to(DEV), dense["values"][i][h // G].to(DEV)
            s = q[row:row + new, h].double() @ keys.T / 8
            pos = torch.arange(length - new, length)[:, None]
            seen = ((torch.arange(length) <= pos) & keep).to(DEV)
            p = torch.where(seen, (s - s.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True).clamp(min=-1e300)).exp(), 0.0)
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            err = (got[row:row + new, h].double() - p @ values).abs()
            assert bool((err <= 2.0 ** -8 * (p @ values).abs() + 2.0 ** -9 * (p @ values.abs())).all())
        row += new


@gpu
@pytest.mark.parametrize("new", [1, 90])
def test_extreme_queries_and_scales(new):
    """Rows of bf16 beyond fp16's range, rows of zeros, infinite and NaN rows beside ordinary ones; blocks of values that are
    nearly zero beside large ones, with the weight on them."""
    lengths, H, D = [200], 1, 128
    cache, table, dense = _filled(lengths, H, D, 16, "int8", 17)
    small = table[0, 3:6].long()
    cache.value_scales[small] *= 1e-20
    for b in (3, 4, 5):
        dense["values"][0][:, 16 * b:16 * b + 16] *= float(np.float32(1e-20))
    q = torch.randn(new, 6, D, generator=torch.Generator().manual_seed(9)).to(DEV)
    q[:, 0] *= 0
    q[:, 1] *= 1e-30
    q[:, 2] = 8 * dense["keys"][0][0, 70].to(DEV).float()          # all weight on a token whose values are nearly zero
    q[:, 3, :5] = 0
    q = q.bfloat16()
    scale = 0.05
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got, lse = cache.attend(q, table.to(DEV), lens, scale=scale, lse=True)
    _check_attend(q, got, None, dense, lengths, [new], 0, scale)
    assert torch.isfinite(got).all() and torch.isfinite(lse).all()
    big = q.clone()
    big[:, 4] *= 2.0 ** 60
    big[:, 0, 0], big[:, 1, 7] = math.nan, math.inf
    other = cache.attend(big, table.to(DEV), lens, scale=scale)
    assert torch.isnan(other[:, 0]).all() and torch.isnan(other[:, 1]).all()
    assert torch.equal(other[:, [2, 3, 5]], got[:, [2, 3, 5]])
    assert torch.isfinite(other[:, 4]).all()
    scaled = cache.attend((q.float() * 2.0 ** 40).bfloat16(), table.to(DEV), lens, scale=scale * 2.0 ** -40)
    assert torch.equal(scaled[:, [0, 2, 3, 4, 5]], got[:, [0, 2, 3, 4, 5]])


@gpu
@pytest.mark.parametrize("new,G", [(1, 4), (130, 2)])
def test_attention_and_append_replay_from_a_graph_with_other_lengths(new, G):
    lengths, H, D, T = [400, 410], 2, 64, 64
    cache, table, dense = _filled(lengths, H, D, T, "int8", 19, width=9)
    q = torch.randn(2 * new, H * G, D, generator=torch.Generator().manual_seed(3)).half().to(DEV)
    k = torch.randn(2 * new, H, D, generator=torch.Generator().manual_seed(4)).half().to(DEV)
    table, lens = table.to(DEV), torch.tensor([new + 1, new + 5], dtype=torch.int32, device=DEV)
    twin = jq.KVCache(*(getattr(cache, n).clone() for n in ("keys", "values", "key_scales", "value_scales")), "int8")
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        cache.attend(q, table, lens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            cache.append(k, k, table, lens)
            out = cache.attend(q, table, lens)
    for n in (350, 399, 400):
        lens.copy_(torch.tensor([n, n + 10], dtype=torch.int32))
        graph.replay()
        twin.append(k, k, table, lens)
        want = twin.attend(q, table, lens)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(cache.keys, twin.keys)


APPEND = [
    # lengths after, new, heads, D, T, format, dtype
    ([1], [1], 1, 32, 16, "int8", torch.float32),
    ([16, 17, 33, 40], [1, 1, 17, 40], 3, 64, 16, "e4m3", torch.bfloat16),
    ([64, 65, 130, 0, 90], [64, 1, 129, 0, 30], 2, 128, 64, "int8", torch.bfloat16),
    ([300, 257], [2, 200], 2, 96, 128, "e4m3", torch.float16),
    ([100, 7], [33, 7], 1, 256, 32, "int8", torch.float16),
    ([45, 46], [9, 9], 2, 160, 16, "e4m3", torch.float32),
]


@gpu
@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}-{c[5]}")
@pytest.mark.parametrize("values", ["usual", "growing", "odd"])
def test_append_and_read_bit_for_bit(case, values):
    lengths, new, H, D, T, fmt, dtype = case
    cache, table, _ = _filled(lengths, H, D, T, fmt, sum(lengths) + D)
    gen = torch.Generator().manual_seed(1)
    n = sum(new)
    k, v = torch.randn(n, H, D, generator=gen) * 0.02, torch.randn(n, H, D, generator=gen) * 3
    if values == "growing":
        k, v = k * 1e4, v * 1e-30
    if values == "odd":
        k[::3, :, 1], k[::5, :, 2], k[1::4] = math.nan, -math.inf, 0
        v[:, :, 3], v[::2] = math.inf, -0.0
    k, v = k.to(dtype), v.to(dtype)
    before = {w: getattr(cache, w).cpu().numpy().reshape(cache.blocks, H, T * D).copy() for w in ("keys", "values")}
    scales = {w: getattr(cache, w[:-1] + "_scales").cpu().numpy().copy() for w in ("keys", "values")}
    lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    cache.append(k.to(DEV), v.to(DEV), table.to(DEV), lens, _starts(new).to(DEV), max_new=max(new))
    read = dict(zip(("keys", "values"), cache.read(table.to(DEV), lens, max(lengths) + 5)))
    half = dict(zip(("keys", "values"), cache.read(table.to(DEV), lens, 5, torch.bfloat16)))
    for what, x in (("keys", k), ("values", v)):
        place = oracle.places(T, D, what)
        want = read[what].new_zeros(read[what].shape).cpu().numpy()
        row = 0
        defined = np.zeros((cache.blocks, T), bool)
        for i, (length, m) in enumerate(zip(lengths, new)):
            first = length - m
            for b in range(-(-length // T)):
                at = int(table[i, b])
                held = min(max(first - b * T, 0), T)
                end = min(length - b * T, T)
                defined[at, :end] = True
                for h in range(H):
                    codes = before[what][at, h][place]
                    if end > held:
                        fresh = x[row + b * T + held - first:row + b * T + end - first, h].float().numpy()
                        codes, scales[what][at, h] = oracle.append_block(codes, scales[what][at, h], held, fresh, fmt)
                    before[what][at, h][place[:end]] = codes[:end]
                    want[i, want.shape[1] - length + b * T:want.shape[1] - length + b * T + end, h] = \
                        oracle.decode(codes[:end], fmt) * scales[what][at, h]
            row += m
        after = getattr(cache, what).cpu().numpy().reshape(cache.blocks, H, T * D)
        for at in range(cache.blocks):
            used = place[defined[at]].reshape(-1)
            assert np.array_equal(after[at][:, used], before[what][at][:, used])
        assert np.array_equal(getattr(cache, what[:-1] + "_scales").cpu().numpy(), scales[what])
        assert np.array_equal(read[what].cpu().numpy(), want)
        assert torch.equal(half[what].cpu(), torch.from_numpy(want[:, -5:]).bfloat16())


@gpu
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_quotients_near_the_middle_of_two_codes(fmt):
    """Values at and beside every boundary between two codes, for scales of many mantissas: the kernel's product with the
    reciprocal has to end where the quotient does."""
    H, D, T = 64, 128, 128
    cache = jq.KVCache.empty(1, H, D, block_size=T, fmt=fmt, device=DEV)
    gen = torch.Generator().manual_seed(2)
    grid = oracle.e4m3_values()[:127] if fmt == "e4m3" else np.arange(128.0)
    middle = (grid[1:] + grid[:-1]) / 2
    x = torch.empty(T, H, D)
    for h in range(H):
        top = np.float32(np.exp(torch.randn((), generator=gen).item() * 20))
        scale = np.float32(top / oracle.TOP[fmt])
        near = (middle * float(scale)).astype(np.float32)
        steps = torch.randint(-6, 7, (T, D), generator=gen).numpy().astype(np.int32)
        pick = torch.randint(0, len(near), (T, D), generator=gen).numpy()
        x[:, h] = torch.from_numpy((near[pick].view(np.int32) + steps).view(np.float32) * np.sign(steps + 0.5).astype(np.float32)).clamp(-float(top), float(top))
        x[0, h, 0] = float(top)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.tensor([T], dtype=torch.int32, device=DEV)
    cache.append(x.to(DEV), -x.to(DEV), table, lens)
    got = cache.keys.cpu().numpy().reshape(H, T * D), cache.values.cpu().numpy().reshape(H, T * D)
    for h in range(H):
        for what, codes, sign in (("keys", got[0], 1), ("values", got[1], -1)):
            want, _ = oracle.append_block(np.zeros((T, D), np.uint8), 0, 0, sign * x[:, h].numpy(), fmt)
            assert np.array_equal(codes[h][oracle.places(T, D, what)], want)


@gpu
def test_more_prompts_than_are_planned_at_once():
    """2500 short prompts: over 32 segments for every CTA of the prompt kernel; and more new tokens than max_new names (tokens beyond it
    may be left out by append, and nothing else happens)."""
    S, H, D, T, new = 2500, 2, 64, 64, 33
    lengths = [new + i % 32 for i in range(S)]
    cache, table, dense = _filled(lengths, H, D, T, "int8", 5)
    q = torch.randn(S * new, H, D, generator=torch.Generator().manual_seed(6)).half().to(DEV)
    table, lens = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    got = cache.attend(q, table, lens)
    for i in range(0, S, 83):
        _check_attend(q[i * new:(i + 1) * new], got[i * new:(i + 1) * new], None, {k: [v[i]] for k, v in dense.items()}, [lengths[i]], [new], 0)
    assert torch.isfinite(got).all()
    starts = _starts([new] * S).to(DEV)
    for few in (1, 3, 40):                                     # any max_new gives every query its output
        assert torch.isfinite(cache.attend(q, table, lens, starts, max_new=few)).all()
    keys = cache.keys.clone()
    k = torch.randn(S * new, H, D, device=DEV)
    cache.append(k, k, table, lens, starts, max_new=5)
    changed = (cache.keys != keys).view(cache.blocks, -1).any(1)
    assert changed.any() and ops.check_status(raise_on_error=False) == 0


@gpu
def test_append_writes_nothing_where_the_table_names_nothing():
    cache, table, _ = _filled([100, 60], 2, 64, 16, "int8", 3)
    keys, scales = cache.keys.clone(), cache.key_scales.clone()
    k = torch.randn(160, 2, 64, device=DEV)
    lens = torch.tensor([100, 60], dtype=torch.int32, device=DEV)
    bad = torch.full_like(table, -1)
    bad[1] = cache.blocks
    cache.append(k, k, bad.to(DEV), lens, _starts([100, 60]).to(DEV))
    for starts in ([-3, 5, 9], [0, 200, 161], [5, 2, 1]):           # rows that the call does not have
        cache.append(k, k, table.to(DEV), lens, torch.tensor(starts, dtype=torch.int32, device=DEV), max_new=100)
        if starts[1] == 5:
            assert torch.isfinite(cache.attend(k.half(), table.to(DEV), lens, torch.tensor(starts, dtype=torch.int32, device=DEV), max_new=100)[5:9]).all()
            cache.keys.copy_(keys)
            cache.key_scales.copy_(scales)
    assert torch.equal(cache.keys, keys) and torch.equal(cache.key_scales, scales)
    cache.append(k[:0], k[:0], table.to(DEV), lens)
    assert cache.attend(k[:0].half(), table.to(DEV), lens).shape == (0, 2, 64)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert cache.attend(k[:0].half(), table[:0].to(DEV), none).shape == (0, 2, 64)
    got = cache.read(table.to(DEV), lens, 0)
    assert got[0].shape == (2, 0, 2, 64)


def _host_cache(**over):
    c = _lib.jq_kv_cache(1 << 20, 1 << 20, 1 << 20, 1 << 20, 4, 2, 64, 16, 0, 0)
    b = _lib.jq_kv_batch(1 << 20, 1 << 20, None, 2, 3, 3, 4, 0, 0)
    for name, value in over.items():
        setattr(c if hasattr(c, name) else b, name, value)
    return c, b


@pytest.mark.parametrize("over,status", [
    (dict(keys=0), -1), (dict(value_scales=0), -1), (dict(table=0), -1), (dict(lengths=0), -1),
    (dict(fmt=2), -4), (dict(block_size=24), -2), (dict(head_dim=40), -2), (dict(head_dim=288), -2), (dict(blocks=0), -2),
    (dict(kv_heads=0), -2), (dict(sequences=-1), -2), (dict(sequences=3), -2), (dict(table_width=0), -2), (dict(table_stride=2), -2),
    (dict(tokens=-1), -2), (dict(keys=(1 << 20) + 8), -3), (dict(key_scales=(1 << 20) + 2), -3), (dict(starts=(1 << 20) + 1), -3),
    (dict(table_width=1 << 28, table_stride=1 << 28), -2),
])
def test_the_library_refuses_on_the_host(over, status):
    lib, (c, b) = _lib.load(), _host_cache(**over)
    import ctypes
    st, p, r = (ctypes.c_int64 * 2)(128, 64), 1 << 20, ctypes.byref
    assert lib.jq_kv_append(r(c), r(b), p, p, st, st, 0, None) == status
    assert lib.jq_kv_read(r(c), r(b), 3, p, p, 0, None) == status
    assert lib.jq_kv_attend(r(c), r(b), p, st, 4, 0.1, 0, p, None, 1, p, 1 << 40, None) == status
    assert lib.jq_kv_attend_workspace_bytes(r(c), r(b), 4) == 0


def test_the_library_refuses_arguments_of_a_call():
    import ctypes
    lib, (c, b) = _lib.load(), _host_cache()
    st, p, r = (ctypes.c_int64 * 2)(128, 64), 1 << 20, ctypes.byref
    assert lib.jq_kv_append(None, r(b), p, p, st, st, 0, None) == -1
    assert lib.jq_kv_append(r(c), r(b), None, p, st, st, 0, None) == -1
    assert lib.jq_kv_append(r(c), r(b), p, p, st, st, 3, None) == -4
    assert lib.jq_kv_append(r(c), r(b), p + 1, p, st, st, 2, None) == -3
    assert lib.jq_kv_read(r(c), r(b), -1, p, p, 0, None) == -2
    assert lib.jq_kv_read(r(c), r(b), 3, p + 4, p, 0, None) == -3
    attend = lambda q=p, heads=4, scale=0.1, window=0, out=p, dtype=1, ws=p, size=1 << 40, cache=c: lib.jq_kv_attend(      # noqa: E731
        r(cache), r(b), q, st, heads, scale, window, out, None, dtype, ws, size, None)
    assert attend(q=None) == -1 and attend(out=None) == -1 and attend(ws=None) == -1
    assert attend(heads=3) == -2 and attend(heads=0) == -2 and attend(window=-1) == -2
    assert attend(scale=0.0) == -2 and attend(scale=-1.0) == -2 and attend(scale=math.nan) == -2 and attend(scale=math.inf) == -2
    assert attend(dtype=0) == -4 and attend(q=p + 1) == -3 and attend(out=p + 8) == -3 and attend(ws=p + 16) == -3
    assert attend(size=1024) == -6
    assert attend(cache=_host_cache(head_dim=96)[0]) == -5


def test_the_python_layer_refuses():
    cache = jq.KVCache.empty(4, 2, 64, block_size=16, device="cpu")
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.float16)
    assert cache.nbytes() == 2 * 4 * 2 * 16 * 64 + 2 * 4 * 2 * 4
    for call, text in (
            (lambda: cache.attend(q, table, lens), "CUDA"),
            (lambda: cache.append(q[:, :2], q[:, :2], table, lens), "CUDA"),
            (lambda: cache.read(table, lens, 3), "CUDA"),
            (lambda: cache.attend(q.float(), table, lens), "query dtype"),
            (lambda: cache.attend(q[:, :3], table, lens), "key heads"),
            (lambda: cache.attend(q[..., :32], table, lens), "key heads"),
            (lambda: cache.attend(q, table.long(), lens), "int32"),
            (lambda: cache.attend(q, table[:1], lens), "sequences"),
            (lambda: cache.attend(q[:1], table, lens), "starts"),
            (lambda: cache.attend(q, table, lens, lens), "starts"),
            (lambda: cache.attend(q, table[:, :0], lens), "columns"),
            (lambda: cache.attend(q, table.t()[:2], lens), "contiguous"),
            (lambda: cache.attend(q, table, lens, scale=0.0), "scale"),
            (lambda: cache.attend(q, table, lens, window=-1), "window"),
            (lambda: cache.attend(q, table, lens, max_new=-1), "max_new"),
            (lambda: cache.append(q, q, table, lens), "2, 64"),
            (lambda: cache.append(q[:, :2], q[:, 2:].float(), table, lens), "one shape"),
            (lambda: cache.append(q[:, :2].double(), q[:, :2].double(), table, lens), "dtype"),
            (lambda: cache.read(table, lens, -1), "last"),
            (lambda: jq.KVCache.empty(4, 2, 96, device="cpu").attend(torch.zeros(2, 4, 96).half(), table, lens), "heads of"),
    ):
        with pytest.raises(RuntimeError, match=text):
            call()
    keys = cache.keys
    for args in ((keys, keys, cache.key_scales, cache.value_scales, "fp8"), (keys[0], keys, cache.key_scales, cache.value_scales),
                 (keys, keys, cache.key_scales.half(), cache.value_scales), (keys[:, :, :8], keys[:, :, :8], cache.key_scales, cache.value_scales),
                 (keys[..., ::2], keys[..., ::2], cache.key_scales, cache.value_scales)):
        with pytest.raises(ValueError):
            jq.KVCache(*args)
    with pytest.raises(ValueError):
        jq.KVCache.empty(4, 2, 48, device="cpu")


TENSORS = ("keys", "values", "key_scales", "value_scales")


def _through_a_file(cache):
    file = io.BytesIO()
    torch.save(cache, file)
    file.seek(0)
    return torch.load(file, weights_only=False)


def _replaced(cache):
    other = copy.copy(cache)
    for name in TENSORS:
        setattr(other, name, getattr(cache, name).clone())
    return other


def _replaced_in_place(cache):
    other = jq.KVCache(*(getattr(cache, name)[:1].clone() for name in TENSORS), cache.fmt)
    for name in TENSORS:
        getattr(other, name).data = getattr(cache, name).clone()
    return other


COPIES = [copy.deepcopy, _through_a_file, _replaced, _replaced_in_place]


@pytest.mark.parametrize("make", COPIES)
def test_a_copy_names_its_own_memory(make):
    cache = jq.KVCache.empty(5, 2, 64, block_size=16, fmt="e4m3", device="cpu")
    other = make(cache)
    for c in (cache, other):
        seen = _lib.jq_kv_cache.from_buffer_copy(c._structure())
        assert [seen.keys, seen.values, seen.key_scales, seen.value_scales] == [getattr(c, name).data_ptr() for name in TENSORS]
        assert (seen.blocks, seen.kv_heads, seen.head_dim, seen.block_size, seen.fmt) == (5, 2, 64, 16, _lib.JQ_KV_E4M3)
        assert (c.blocks, c.kv_heads, c.head_dim, c.block_size) == (5, 2, 64, 16)
    assert all(getattr(cache, name).data_ptr() != getattr(other, name).data_ptr() for name in TENSORS)


def test_replaced_tensors_are_looked_over():
    cache = jq.KVCache.empty(5, 2, 64, block_size=16, device="cpu")
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    for name, value in (("keys", torch.zeros(5, 2, 16, 64)), ("value_scales", torch.ones(4, 2)), ("fmt", "fp8"), ("values", cache.values[:, :, :8])):
        other = copy.copy(cache)
        setattr(other, name, value)
        with pytest.raises(ValueError):
            other.read(table, lens, 3)
    cache.keys.data = cache.keys[:3].clone()
    with pytest.raises(ValueError):
        cache.read(table, lens, 3)
    cache.values, cache.key_scales, cache.value_scales = cache.values[:3].clone(), cache.key_scales[:3].clone(), cache.value_scales[:3].clone()
    assert _lib.jq_kv_cache.from_buffer_copy(cache._structure()).blocks == cache.blocks == 3


@gpu
@pytest.mark.parametrize("make", COPIES)
def test_a_copy_appends_and_attends_to_its_own_memory(make):
    lengths, H, D = [100, 60], 2, 64
    cache, table, dense = _filled(lengths, H, D, 16, "int8", 21)
    kept = [getattr(cache, name).clone() for name in TENSORS]
    other = make(cache)
    table, lens = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    q = torch.randn(2, 4, D, device=DEV).half()
    _check_attend(q, other.attend(q, table, lens), None, dense, lengths, [1, 1], 0)
    k = torch.randn(2, H, D, device=DEV)
    other.append(k, k, table, lens)
    assert all(torch.equal(getattr(cache, name), was) for name, was in zip(TENSORS, kept))
    assert not torch.equal(other.keys, cache.keys)
    twin = jq.KVCache(*kept, "int8")
    twin.append(k, k, table, lens)
    assert all(torch.equal(getattr(other, name), getattr(twin, name)) for name in TENSORS)
    want = twin.attend(q, table, lens)
    del cache, twin, kept
    assert torch.equal(other.attend(q, table, lens), want)
    assert all(torch.equal(a, b) for a, b in zip(other.read(table, lens, 60), make(other).read(table, lens, 60)))


def test_captured_calls_have_a_status_word_that_is_read(monkeypatch):
    """What a captured call is given as its status word is what check_status() reads, and not a place in the graph's memory."""
    lib, words = _lib.load(), {4096: -7}
    monkeypatch.setattr(lib, "jq_status_word", lambda: 4096)
    monkeypatch.setattr(lib, "jq_ta_status", lambda at, clear, stream: words.pop(at, 0))
    monkeypatch.setattr(ops, "_capturing", lambda stream: True)
    monkeypatch.setattr(ops, "_stream", lambda: 7)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: type("Stream", (), {"cuda_stream": 7}))
    own, at, size, status = ops._parts_workspace(torch.device("cpu"), 8192, 7)
    assert own.data_ptr() == at and size == 8192 and bool((own[:ops._PARTS_DATA] == 0).all())
    assert status == 4096
    with pytest.raises(_lib.JqError):
        ops.check_status()
    assert ops.check_status() == 0


@gpu
@pytest.mark.parametrize("new", [1, 90])
def test_a_wait_that_gives_up_in_a_replay_is_seen(new, monkeypatch):
    """The word is raised as a kernel would raise it, by a wait that runs out; neither the graph's own zeroing nor what is captured
    behind the call may clear it, and it is seen on a stream that the graph was not captured on."""
    lengths, H, D = [300, 150], 2, 64
    cache, table, _ = _filled(lengths, H, D, 32, "int8", 23)
    q = torch.randn(2 * new, 4, D, device=DEV).half()
    table, lens = table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = cache.attend(q, table, lens)
    lib, given = _lib.load(), []
    real = lib.jq_kv_attend_status
    monkeypatch.setattr(lib, "jq_kv_attend_status", lambda *a: given.append(a[-2]) or real(*a))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, table, lens)
        behind = [torch.zeros(1 << 20, dtype=torch.uint8, device=DEV) + 1 for _ in range(4)]
    graph.replay()
    assert torch.equal(out, want) and ops.check_status(raise_on_error=False) == 0
    assert given[0] and lib.jq_selftest_bounded_wait(given[0], 4096, None) == 0
    graph.replay()
    assert torch.equal(out, want) and all(bool((b == 1).all()) for b in behind)
    with pytest.raises(_lib.JqError):
        ops.check_status()
    assert ops.check_status() == 0


FIRST = """
import sys
import torch
sys.path.insert(0, sys.argv[1])
import if_i_could_turn_back_time_b200 as jq
from if_i_could_turn_back_time_b200 import ops
cache = jq.KVCache.empty(8, 2, 64, block_size=16)
table = torch.arange(8, dtype=torch.int32, device="cuda").view(1, 8)
lens = torch.tensor([100], dtype=torch.int32, device="cuda")
q = torch.randn(1, 4, 64, device="cuda").half()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = cache.attend(q, table, lens)
graph.replay()
assert ops.check_status() == 0 and bool((out == 0).all())
print("captured")
"""


@gpu
def test_a_capture_that_is_the_librarys_first_call():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST, root], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "captured", r.stderr[-2000:]


def test_tokens_of_no_sequence_are_refused():
    """Nothing would be written for them: the outputs would be what the memory held."""
    import ctypes
    lib, (c, b) = _lib.load(), _host_cache(sequences=0, tokens=4)
    st, p, r = (ctypes.c_int64 * 2)(128, 64), 1 << 20, ctypes.byref
    for starts in (None, p):
        b.starts = starts
        assert lib.jq_kv_append(r(c), r(b), p, p, st, st, 0, None) == -2
        assert lib.jq_kv_attend(r(c), r(b), p, st, 4, 0.1, 0, p, None, 1, p, 1 << 40, None) == -2
        assert lib.jq_kv_attend_workspace_bytes(r(c), r(b), 4) == 0
    b.tokens = 0
    assert lib.jq_kv_append(r(c), r(b), p, p, st, st, 0, None) == 0
    cache = jq.KVCache.empty(4, 2, 64, block_size=16, device="cpu")
    table, lens, q = torch.zeros(0, 3, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(2, 4, 64).half()
    for starts in (None, torch.zeros(1, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="no sequence"):
            cache.attend(q, table, lens, starts)
        with pytest.raises(RuntimeError, match="no sequence"):
            cache.append(q[:, :2], q[:, :2], table, lens, starts)


@gpu
def test_a_refused_call_leaves_no_workspace_size_behind():
    """A table of more tokens than positions have bits is refused by the library; the same heads and tokens with another table are not."""
    cache = jq.KVCache.empty(4, 2, 64, block_size=128, device=DEV)
    q = torch.zeros(1, 8, 64, device=DEV).half()
    lens = torch.tensor([100], dtype=torch.int32, device=DEV)
    with pytest.raises(_lib.JqError):
        cache.attend(q, torch.zeros(1, 1 << 24, dtype=torch.int32, device=DEV), lens)
    assert not cache._need
    assert bool((cache.attend(q, torch.zeros(1, 1, dtype=torch.int32, device=DEV), lens) == 0).all())


def test_counts_past_32_bits():
    """A max_new that is larger than the call stands for all its tokens; what the library cannot count is refused."""
    cache = jq.KVCache.empty(4, 2, 64, block_size=16, device="cpu")
    cache._cuda = True                                  # (nothing is called)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    assert _lib.jq_kv_batch.from_buffer_copy(cache._batch(table, lens, None, 6, 1 << 40)).max_new == 6
    with pytest.raises(RuntimeError, match="32 bits"):
        cache._batch(table, lens, None, 1 << 32, 5)
    with pytest.raises(RuntimeError, match="last"):
        cache.read(table, lens, 1 << 32)


@gpu
@pytest.mark.parametrize("new,G", [(1, 2), (5, 4), (40, 2)])
@pytest.mark.parametrize("fmt,D", [("int8", 64), ("e4m3", 128)])
def test_blocks_before_every_window_may_hold_anything(new, G, fmt, D):
    """A sequence's blocks that no window reaches any more are another's, who has not filled them: codes and scales that are NaN."""
    lengths, H, T, window = [320, 450], 2, 16, 100
    cache, table, dense = _filled(lengths, H, D, T, fmt, 29)
    bad = [b for b in range(cache.blocks) if b not in set(table.flatten().tolist())][0]
    for what in ("keys", "values"):
        getattr(cache, what)[bad] = 0x7F if fmt == "e4m3" else 0
        getattr(cache, what[:-1] + "_scales")[bad] = math.nan
    for i, length in enumerate(lengths):
        first = length - new - window + 1
        assert first % 64 >= 16                                    # (whole blocks before it in the 64 keys that it lies in)
        table[i, :first // T] = bad
    q = torch.randn(2 * new, H * G, D, generator=torch.Generator().manual_seed(9)).bfloat16().to(DEV)
    got, lse = cache.attend(q, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window, lse=True)
    _check_attend(q, got, lse, dense, lengths, [new] * 2, window)


@gpu
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("power", [120, -118])
def test_queries_at_the_ends_of_their_type(new, power):
    """Rows of bf16 whose largest value is near 2^123 or below 2^-116, with a scale that brings the scores back."""
    lengths, H, D = [200], 1, 128
    cache, table, dense = _filled(lengths, H, D, 16, "int8", 17)
    q = torch.randn(new, 6, D, generator=torch.Generator().manual_seed(9)).mul(1.5 * 2.0 ** power).bfloat16().to(DEV)
    got, lse = cache.attend(q, table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=0.05 * 2.0 ** -power, lse=True)
    _check_attend(q, got, lse, dense, lengths, [new], 0, 0.05 * 2.0 ** -power)


@gpu
@pytest.mark.parametrize("new", [1, 90])
def test_keys_of_zeros_and_queries_of_nearly_zero(new):
    """The factor of the scores (2^-67 of the keys' scale, 2^-113 of the query's) has no fp32 number: every visible key weighs the same."""
    length, H, D = 150, 1, 64
    cache = jq.KVCache.empty(10, H, D, block_size=16, device=DEV)
    table, lens = torch.arange(10, dtype=torch.int32, device=DEV)[None], torch.tensor([length], dtype=torch.int32, device=DEV)
    gen = torch.Generator().manual_seed(9)
    cache.append(torch.zeros(length, H, D, device=DEV), torch.randn(length, H, D, generator=gen).to(DEV), table, lens)
    k, v = cache.read(table, lens, length)
    q = torch.randn(new, 3, D, generator=gen).mul(1e-30).bfloat16().to(DEV)
    got, lse = cache.attend(q, table, lens, lse=True)
    _check_attend(q, got, lse, {"keys": [k[0].transpose(0, 1).double()], "values": [v[0].transpose(0, 1).double()]}, [length], [new], 0)


@gpu
@pytest.mark.parametrize("new,D,fmt", [(1, 64, "int8"), (1, 128, "e4m3"), (5, 128, "int8"), (40, 64, "e4m3"), (40, 128, "int8")])
def test_one_strong_token_before_a_long_text(new, D, fmt):
    """An attention sink: the first token has nearly all the weight and a value that is nearly zero, so that what counts is the sum of
    thousands of small weights.  The bound is the module's with 2^-32 of the largest weight in place of 2^-25 for those that are not rounded
    to eleven bits, and fp32 sums of one term for 64 keys.  More sequences share the text than there are CTAs: one alone would be cut
    into parts, with the strong token in one of them."""
    length, T, H, S, gaps = 16384, 64, 1, 600 if new < 10 else 160, [11.0, 13.2, 14.284, 15.2, 16.1]
    blocks = length // T
    gen = torch.Generator().manual_seed(31)
    top = 127.0 if fmt == "int8" else 448.0
    keys, values = torch.zeros(blocks, T, D), torch.randint(64, 113, (blocks, T, D), generator=gen).float()
    keys[0, 0, 0], values[0, 0] = top, 1.0
    cache = jq.KVCache.empty(blocks, H, D, block_size=T, fmt=fmt, device=DEV)
    dense = {}
    for what, x in (("keys", keys), ("values", values)):
        codes = x.add(128).to(torch.uint8) if fmt == "int8" else x.to(torch.float8_e4m3fn).view(torch.uint8)
        laid = torch.empty(blocks, T * D, dtype=torch.uint8)
        laid[:, torch.from_numpy(oracle.places(T, D, what).reshape(-1))] = codes.reshape(blocks, T * D)
        getattr(cache, what).copy_(laid.view(blocks, H, T, D))
        getattr(cache, what[:-1] + "_scales").fill_(2.0 ** -6)
        real = torch.from_numpy(oracle.decode(codes.numpy(), fmt)).double() * 2.0 ** -6
        dense[what] = real.reshape(length, D).to(DEV)
    q = torch.zeros(new, len(gaps), D)
    q[:, :, 0] = torch.tensor(gaps) / (top * 2.0 ** -6)
    q = q.half().to(DEV)
    table, lens = torch.arange(blocks, dtype=torch.int32, device=DEV).expand(S, blocks).contiguous(), torch.full((S,), length, dtype=torch.int32, device=DEV)
    got, lse = cache.attend(q.expand(S, new, len(gaps), D), table, lens, scale=1.0, lse=True)
    for h in range(len(gaps)):
        ref, want, weight, size = oracle.attend(q[:, h], dense["keys"], dense["values"], length - new, 1.0, 0)
        off = D * 2.0 ** -24 * size + 2.0 ** -23 * size + 2.0 ** -21 + length / 64 * 2.0 ** -24
        bound = (2.0 ** -11 + 2 * off)[:, None] * weight + 2.0 ** -32 * length * dense["values"].max() + 2.0 ** -11 * ref.abs() + 2.0 ** -24
        err = (got[:, :, h].double() - ref).abs().amax(0)
        assert bool((err <= bound).all()), (gaps[h], (err / bound).max().item(), (err / ref).max().item())
        assert bool(((lse[:, :, h].double() - want).abs() <= off + 2.0 ** -22 * want.abs()).all())


@gpu
@pytest.mark.parametrize("pairs", ["few", "many"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("D,new,G", [(64, 1, 7), (64, 3, 5), (64, 2, 9), (64, 9, 3), (64, 4, 8), (128, 2, 4), (128, 1, 16), (128, 8, 3), (128, 2, 9)])
def test_every_tile_of_few_rows(D, new, G, fmt, pairs):
    """Up to 24 rows (32 at 64 values) of a key head go through one kernel in tiles of 8, 16, 24 or 32 rows, with wide CTAs where pairs of a
    sequence and a key head are at most half as many as SMs, with narrow ones where they are more."""
    S, H = (5, 2) if pairs == "few" else (24, 4)
    gen = torch.Generator().manual_seed(D + new + G)
    lengths = [1 + (37 * i * i + 11 * i) % 400 for i in range(S)]
    lengths[1], lengths[3] = 0, 1500
    news = [max(0, new - i % 3) if i else new for i in range(S)]
    cache, table, dense = _filled(lengths, H, D, 32 if G > 5 else 16, fmt, 37)
    q = torch.randn(sum(news), H * G, D, generator=gen).mul(1.5).to(torch.float16 if G % 2 else torch.bfloat16).to(DEV)
    args = (table.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), _starts(news).to(DEV), new)
    for window in (0, 130):
        got, lse = cache.attend(q, *args, window=window, lse=True)
        _check_attend(q, got, lse, dense, lengths, news, window)
        assert torch.equal(cache.attend(q, *args, window=window), got)
    assert ops.check_status(raise_on_error=False) == 0


@pytest.mark.parametrize("scale", [2.5e38, 3e38, 1e-50])
def test_scales_that_fp32_cannot_hold_are_refused(scale):
    """(2.5e38 log2(e) is infinite: every output would be NaN.)"""
    import ctypes
    lib, (c, b) = _lib.load(), _host_cache()
    st, p, r = (ctypes.c_int64 * 2)(128, 64), 1 << 20, ctypes.byref
    assert lib.jq_kv_attend(r(c), r(b), p, st, 4, scale, 0, p, None, 1, p, 1024, None) == -2
    cache = jq.KVCache.empty(4, 2, 64, block_size=16, device="cpu")
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.tensor([5, 9], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="scale"):
        cache.attend(torch.zeros(2, 4, 64).half(), table, lens, scale=scale)


class Layered(jq.KVCache):
    def __init__(self, layer):
        empty = jq.KVCache.empty(3, 2, 64, block_size=16, device="cpu")
        super().__init__(*(getattr(empty, name) for name in TENSORS))
        self.layer = layer


@pytest.mark.parametrize("make", [copy.copy, copy.deepcopy, _through_a_file])
def test_a_copy_is_what_the_cache_is(make):
    other = make(Layered(7))
    assert type(other) is Layered and other.layer == 7 and other.nbytes() == Layered(7).nbytes()
    seen = _lib.jq_kv_cache.from_buffer_copy(other._c)
    assert [seen.keys, seen.values, seen.key_scales, seen.value_scales] == [getattr(other, name).data_ptr() for name in TENSORS]
