"""pbmoe_mla_q4_decode where a CTA of the attention walks many tiles: long
splits, a maximum that moves inside one, weights far apart.

The planner takes the fewest 64-row tiles a CTA that fill one wave, so short
sequences are one tile a CTA. 128 heads and 32 sequences leave 37 CTAs' worth
of rows a head block: a sequence is then one split of all its tiles. Sequences
may share their buffers, so that a long one need not be stored 32 times.

Outputs are held to the share of their norm that random roundings add up to: a
weight takes two of them to fp16 (p, its product with the scale), 2^-11 / sqrt(3)
at most each, and its score's error is that of Q' in fp16, 2^-11 / sqrt(3) of
the latent part's own deviation, sqrt(128 * 512 * 0.02^2 / 192) = 0.37 of the
queries'. Terms of an output add up in quadrature like the output itself:
4e-4 + 1.1e-4 q_scale, held below 1e-3 + 2^-11 q_scale, and in bf16 below 3e-3
more.
"""

import math

import pytest

import mla_plain as plain

pytestmark = pytest.mark.gpu

NOPE, ROPE, LAT, V = plain.NOPE, plain.ROPE, plain.LAT, plain.V


@pytest.fixture(scope="module")
def ctx():
    import torch

    from pb_b200 import capi

    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    c = capi.Context(0)
    c.mla_q4_reserve(capi.mla_config(heads=128), 32)
    yield c
    c.close()


def _randn(shape, seed, scale=1.0, dtype=None):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or torch.float32)


def _rows(n, seed, mean=0.0):
    import torch

    u, s = plain.quantise(_randn((n, LAT), seed) + mean)
    return plain.pack(u), s, _randn((n, ROPE), seed + 1, dtype=torch.bfloat16)


def _weights(heads, seed=31):
    import torch

    return _randn((heads, NOPE, LAT), seed, 0.02, torch.bfloat16), _randn((heads, V, LAT), seed + 1, 0.02, torch.bfloat16)


def _decode(ctx, rows, lens, q, weights, out_dtype="float32"):
    """rows: one (codes, scales, k_rope) a sequence, or one for all of them."""
    import torch

    from pb_b200 import capi

    rows = rows if isinstance(rows, list) else [rows] * len(lens)
    cache = capi.MlaQ4Cache([r[0] for r in rows], [r[1] for r in rows], [r[2] for r in rows])
    out = torch.empty(len(lens), q.shape[1], V, dtype=getattr(torch, out_dtype), device="cuda")
    ctx.mla_q4_decode(capi.mla_config(heads=q.shape[1]), q, cache, lens, *weights, out)
    return out


def _check(out, rows, lens, q, weights, q_scale, seqs, heads, extra=0.0):
    """Sequences `seqs` and heads `heads` of the outputs against the 64-bit form."""
    import torch

    for b in seqs:
        codes, scales, kr = rows[b] if isinstance(rows, list) else rows
        n = lens[b]
        want = plain.attend_plain(q[b, heads], plain.values(codes[:n], scales[:n]), kr[:n], weights[0][heads],
                                  weights[1][heads])
        assert plain.rms(out[b, heads], want) <= plain.rms_limit(q_scale, out.dtype == torch.bfloat16) + extra, (
            b, n, plain.rms(out[b, heads], want))


@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [200], [1000], [4097], [8000], [30000],
                                  [1, 4097, 15, 16, 17, 8000, 511, 512, 513]])
@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
def test_whole_outputs(ctx, lens, out_dtype):
    rows, w = [_rows(n, 41 + 10 * b) for b, n in enumerate(lens)], _weights(16)
    q = _randn((len(lens), 16, NOPE + ROPE), 33)
    out = _decode(ctx, rows, lens, q, w, out_dtype)
    _check(out, rows, lens, q, w, 1.0, range(len(lens)), slice(None))


@pytest.mark.parametrize("q_scale", [0.0, 0.05, 6.0, 40.0])
def test_score_ranges(ctx, q_scale):
    lens = [2300] * 32
    rows, w = _rows(2300, 71), _weights(128)
    q = _randn((32, 128, NOPE + ROPE), 33, q_scale)
    _check(_decode(ctx, rows, lens, q, w), rows, lens, q, w, q_scale, (0, 31), slice(0, 128, 9))


def test_ragged_batch_of_long_splits(ctx):
    """32 sequences of 1500 to 2500 rows at 128 heads (24 to 40 tiles a CTA), and up to 8192 at 16 heads."""
    lens = [1500 + (b * 331) % 1001 for b in range(32)]
    rows, w = [_rows(n, 100 + 10 * b) for b, n in enumerate(lens)], _weights(128)
    q = _randn((32, 128, NOPE + ROPE), 33)
    _check(_decode(ctx, rows, lens, q, w), rows, lens, q, w, 1.0, (0, 7, 19, 31), slice(0, 128, 11))
    lens = [max(1, (b * 2657) % 8193) for b in range(31)] + [8192]
    rows, w = [_rows(n, 500 + 10 * b) for b, n in enumerate(lens)], _weights(16)
    q = _randn((32, 16, NOPE + ROPE), 33)
    _check(_decode(ctx, rows, lens, q, w), rows, lens, q, w, 1.0, range(32), slice(None))


@pytest.mark.parametrize("bits", [0.25, 2.0, 6.0, 9.0, 13.0, 17.0, 30.0, -0.25, -9.0, -30.0])
def test_scores_that_rise_or_fall_tile_by_tile(ctx, bits):
    """`bits` in base 2 from one 64-row tile to the next, below and beyond what the running maximum may lag."""
    import torch

    n = 1920
    codes, scales, kr = _rows(n, 81)
    kr[:] = 0
    # 64 equal terms: bits * tile = 64 * q * k / sqrt(192) / ln 2, k = tile / 8 a bf16
    kr[:] = (torch.arange(n, device="cuda") // 64 / 8).to(torch.bfloat16).unsqueeze(1)
    q = _randn((32, 128, NOPE + ROPE), 33, 0.3)
    q[..., NOPE:] = bits * math.log(2) * math.sqrt(192) / 8
    rows, lens, w = (codes, scales, kr), [n - 64 * (b % 2) - b for b in range(32)], _weights(128)
    # Q' of the key part as bf16 hi + lo: 2^-17 of scores up to 30 * bits, and as much in their f32 sums
    _check(_decode(ctx, rows, lens, q, w), rows, lens, q, w, 0.3, (0, 31), slice(0, 128, 9),
           extra=30 * abs(bits) * math.log(2) * 2.0**-16)


def test_rows_of_weight_zero_before_low_scores_in_one_split(ctx):
    """Whole tiles that score -inf and then scores far below zero, walked by one CTA: as if the sequence began there."""
    import torch

    n, lost = 640, 192
    codes, scales, kr = _rows(n, 99)
    q = _randn((32, 128, NOPE + ROPE), 34)
    # times the scale in base 2: -1.001, which is not a bf16, so neither half of it is 0
    q[..., NOPE] = -1.001 * math.sqrt(NOPE + ROPE) * math.log(2)
    q[..., NOPE + 1] = -100.0
    kr[:, 0], kr[:, 1] = 0.0, 1000.0
    kr[:lost, 0] = math.inf
    w = _weights(128)
    out = _decode(ctx, (codes, scales, kr), [n] * 32, q, w)
    behind = tuple(x[lost:].contiguous() for x in (codes, scales, kr))
    # the score of -100 * 1000 / sqrt(192) in base 2 is -10412: its f32 sums are off by 2^-11 of a bit, so weights by 2^-11
    _check(out, behind, [n - lost] * 32, q, w, 1.0, (0, 31), slice(0, 128, 9), extra=2.0**-10)


@pytest.mark.parametrize("n,limit", [(32768, 2e-3), (131072, 3e-3)])
def test_long_split_of_random_codes(ctx, n, limit):
    """512 and 2048 tiles in one CTA with nearly equal weights: the output is a sum of n codes of random sign, about
    sqrt(n) of one, while the stored nibbles (8 more each) add up to 8 n. What the f32 sums may lose, when 8 times
    the weights are taken off every four tiles, is 16 steps of 2^-23 of at most 2048 weights' worth: beside sqrt(n) * 2.9
    (the codes' deviation) 2 * 4 * sqrt(n) * 6.6e-7, 1e-3 and 2e-3 at these lengths, on top of the roundings' 1e-3."""
    rows, w = _rows(n, 55), _weights(128)
    q = _randn((32, 128, NOPE + ROPE), 33, 0.02)
    out = _decode(ctx, rows, [n] * 32, q, w)
    heads = slice(0, 128, 17)
    want = plain.attend_plain(q[3, heads], plain.values(rows[0], rows[1]), rows[2], w[0][heads], w[1][heads])
    assert plain.rms(out[3, heads], want) <= limit, plain.rms(out[3, heads], want)


def test_weights_far_below_the_largest_count(ctx):
    """One row that scores 25.5 bits above 2^18 others: together they weigh 0.55% of it. All rows stand for the same
    latent, so the output is that row's: weights lost to fp16 would show as a smaller one."""
    import torch

    n = 1 << 18
    u, s = plain.quantise(_randn((1, LAT), 5) + 1.0)
    codes, scales = plain.pack(u).expand(n, 256).contiguous(), s.expand(n, 8).contiguous()
    kr = torch.zeros(n, ROPE, dtype=torch.bfloat16, device="cuda")
    kr[0] = 4.0
    q = torch.zeros(32, 128, NOPE + ROPE, device="cuda")
    q[..., NOPE:] = 25.5 * math.log(2) * math.sqrt(192) / (64 * 4.0)
    w = _weights(128)
    out = _decode(ctx, (codes, scales, kr), [n] * 32, q, w)
    want = (w[1].double() @ plain.values(codes[:1], scales[:1])[0]).expand(32, 128, V)
    # three fp16 roundings of the one row's weight, all the others' 2^-6 of 0.55% (weights held in 6 bits or more), and
    # the f32 sums: n / 16 MMAs add to one that the first row's weight rules, each truncating it by less than 2^-23 of
    # itself, 2^-9 in all
    assert plain.rms(out, want) <= 3 * plain.F16 + 0.0055 * 2.0**-6 + n / 16 * 2.0**-23


@pytest.mark.parametrize("factor,q_scale", [(2.0**-50, 1.0), (2.0**-20, 1.0), (2.0**20, 0.0), (2.0**98, 0.0)])
def test_scales_over_their_range(ctx, factor, q_scale):
    """Latents from 2^-50 to 2^98 of ordinary ones (the queries' latent part 0 where they are large)."""
    lens, w = [700, 65], _weights(16)
    rows = [(c, (s.float() * factor).bfloat16(), k) for c, s, k in (_rows(n, 91 + n) for n in lens)]
    q = _randn((2, 16, NOPE + ROPE), 33)
    q[..., :NOPE] *= q_scale
    _check(_decode(ctx, rows, lens, q, w), rows, lens, q, w, 1.0, (0, 1), slice(None))
