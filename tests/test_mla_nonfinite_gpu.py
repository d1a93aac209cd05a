"""Latent attention over values that are not finite: what reaches an output as NaN, and what does not."""

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
    c.mla_reserve(capi.mla_config(), 32)
    c.mla_q4_reserve(capi.mla_config(), 32)
    yield c
    c.close()


def _randn(shape, seed, scale=1.0, dtype=None):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or torch.float32)


def _weights():
    import torch

    return _randn((16, NOPE, LAT), 31, 0.02, torch.bfloat16), _randn((16, V, LAT), 32, 0.02, torch.bfloat16)


def _q4_cache(lens, seed):
    import torch

    from pb_b200 import capi

    rows = [plain.quantise(_randn((n, LAT), seed + 10 * b)) for b, n in enumerate(lens)]
    return capi.MlaQ4Cache([plain.pack(u) for u, _ in rows], [s for _, s in rows],
                           [_randn((n, ROPE), seed + 10 * b + 1, dtype=torch.bfloat16) for b, n in enumerate(lens)])


# ------------------------------------------------------------------ 4-bit decode
@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("n", [1, 3, 130, 2000])
def test_q4_decode_nan_scale_reaches_its_whole_sequence(ctx, n, out_dtype):
    import torch

    from pb_b200 import capi

    lens = [100, n, 33]
    cache = _q4_cache(lens, 95)
    wuk, wuv = _weights()
    q = _randn((3, 16, NOPE + ROPE), 33)
    clean, out = (torch.empty(3, 16, V, device="cuda", dtype=getattr(torch, out_dtype)) for _ in range(2))
    ctx.mla_q4_decode(capi.mla_config(), q, cache, lens, wuk, wuv, clean)
    cache.scales[1][n - 1, 2] = math.nan
    ctx.mla_q4_decode(capi.mla_config(), q, cache, lens, wuk, wuv, out)
    assert torch.equal(out[::2], clean[::2]) and bool(clean.isfinite().all())
    assert bool(out[1].isnan().all())


@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
def test_q4_decode_nan_query_reaches_its_whole_head(ctx, out_dtype):
    import torch

    from pb_b200 import capi

    lens = [130, 5]
    cache = _q4_cache(lens, 97)
    wuk, wuv = _weights()
    q = _randn((2, 16, NOPE + ROPE), 33)
    clean, out = (torch.empty(2, 16, V, device="cuda", dtype=getattr(torch, out_dtype)) for _ in range(2))
    ctx.mla_q4_decode(capi.mla_config(), q, cache, lens, wuk, wuv, clean)
    q[0, 3, 7] = math.nan
    q[1, 9, NOPE + 1] = math.inf
    ctx.mla_q4_decode(capi.mla_config(), q, cache, lens, wuk, wuv, out)
    bad = torch.zeros(2, 16, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[1, 9] = True
    assert torch.equal(out[~bad], clean[~bad]) and bool(out[bad].isnan().all())


def test_q4_append_of_a_non_finite_latent_then_decode(ctx):
    """A non-finite latent written by the append latches its bit, and the decode over it says NaN in bf16 too."""
    import torch

    from pb_b200 import capi

    cfg = capi.mla_config()
    ctx.rope_reserve(8192, ROPE, 10000.0)
    cache, pos = capi.MlaQ4Cache.empty(1, 70), torch.arange(70, dtype=torch.int32, device="cuda")
    kv = _randn((70, LAT + ROPE), 3)
    kv[41, 100] = math.inf
    ctx.mla_q4_append(cfg, kv, pos, cache, sequences=torch.zeros_like(pos))
    assert ctx.device_status() == capi.PBMOE_DEV_ERR_CACHE_RANGE
    out = torch.zeros(1, 16, V, device="cuda", dtype=torch.bfloat16)
    q = _randn((1, 16, NOPE + ROPE), 4)
    ctx.mla_q4_decode(cfg, q, cache, [41], *_weights(), out)
    assert bool(out.isfinite().all()) and bool(out.any())
    ctx.mla_q4_decode(cfg, q, cache, [42], *_weights(), out)
    assert bool(out.isnan().all())


# ------------------------------------------------------------------ decode over bf16 rows
@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("what", ["latent", "key"])
def test_decode_nan_row_reaches_its_whole_sequence(ctx, what, out_dtype):
    import torch

    from pb_b200 import capi

    lens, bf = [100, 40, 33], torch.bfloat16
    c, k = [_randn((n, LAT), n, 1.0, bf) for n in lens], [_randn((n, ROPE), n + 1, 1.0, bf) for n in lens]
    wuk, wuv = _weights()
    q = _randn((3, 16, NOPE + ROPE), 33)
    clean, out = (torch.empty(3, 16, V, device="cuda", dtype=getattr(torch, out_dtype)) for _ in range(2))
    ctx.mla_decode(capi.mla_config(), q, c, k, wuk, wuv, clean)
    (c if what == "latent" else k)[1][17, 5] = math.nan
    ctx.mla_decode(capi.mla_config(), q, c, k, wuk, wuv, out)
    assert torch.equal(out[::2], clean[::2]) and bool(out[1].isnan().all())


@pytest.mark.parametrize("out_dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("at", [7, NOPE + 1])
def test_decode_nan_query_reaches_its_whole_head(ctx, at, out_dtype):
    import torch

    from pb_b200 import capi

    lens, bf = [130, 1], torch.bfloat16
    c, k = [_randn((n, LAT), n, 1.0, bf) for n in lens], [_randn((n, ROPE), n + 1, 1.0, bf) for n in lens]
    wuk, wuv = _weights()
    q = _randn((2, 16, NOPE + ROPE), 33)
    clean, out = (torch.empty(2, 16, V, device="cuda", dtype=getattr(torch, out_dtype)) for _ in range(2))
    ctx.mla_decode(capi.mla_config(), q, c, k, wuk, wuv, clean)
    bad = torch.zeros(2, 16, dtype=torch.bool, device="cuda")
    for b, h in ((0, 3), (1, 9)):
        q[b, h, at] = math.nan
        bad[b, h] = True
    ctx.mla_decode(capi.mla_config(), q, c, k, wuk, wuv, out)
    assert torch.equal(out[~bad], clean[~bad]) and bool(out[bad].isnan().all())


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("at", [3, LAT + 6])
def test_append_of_a_nan_then_decode(ctx, at, normed):
    """A NaN latent or key of a token written to bf16 rows, by the append alone and by append + decode."""
    import torch

    from pb_b200 import capi

    cfg, n, bf = capi.mla_config(), 20, torch.bfloat16
    ctx.rope_reserve(8192, ROPE, 10000.0)
    wuk, wuv = _weights()
    norm = torch.ones(LAT, device="cuda") if normed else None
    q, kv = _randn((2, 16, NOPE + ROPE), 3), _randn((2, LAT + ROPE), 4)
    kv[1, at] = math.nan
    pos = torch.full((2,), n - 1, dtype=torch.int32, device="cuda")

    def rows():
        c, k = [_randn((n, LAT), 5 + b, 1.0, bf) for b in range(2)], [_randn((n, ROPE), 7 + b, 1.0, bf) for b in range(2)]
        return c, k, [torch.tensor([t.data_ptr() for t in x], device="cuda") for x in (c, k)]

    c, k, ptrs = rows()
    ctx.mla_rope_append(cfg, q.clone(), kv, pos, *ptrs, n, latent_norm=norm)
    lost = (k if at >= LAT else c)[1][n - 1]
    assert bool(lost.isnan().any()) and bool(lost.isnan().all()) == (normed and at < LAT)
    assert bool(c[0].isfinite().all()) and bool(k[0].isfinite().all())
    c, k, ptrs = rows()
    out = torch.zeros(2, 16, V, device="cuda", dtype=bf)
    ctx.mla_append_decode(cfg, q.clone(), kv, pos, *ptrs, n, c, k, wuk, wuv, out, latent_norm=norm)
    assert ctx.device_status() == 0
    assert bool(out[0].isfinite().all()) and bool(out[1].isnan().all())


# ------------------------------------------------------------------ rows that score -inf everywhere
@pytest.mark.parametrize("n,finite", [(1, 0), (64, 0), (200, 0), (200, 3), (2000, 0), (2000, 1)])
def test_q4_decode_of_infinitely_low_scores(ctx, n, finite):
    """Only -inf scores: NaN, as softmax has it. With `finite` rows at the end: those alone."""
    import torch

    from pb_b200 import capi

    cache = _q4_cache([n], 99)
    q = _randn((1, 16, NOPE + ROPE), 34)
    # times the scale in base 2: -1.001, which is not a bf16, so neither half of it is 0
    q[..., NOPE] = -1.001 * math.sqrt(NOPE + ROPE) * math.log(2)
    kr = cache.k_rope[0]
    kr[:, 0] = 0.0
    kr[:n - finite, 0] = math.inf
    wuk, wuv = _weights()
    out, want = (torch.empty(1, 16, V, device="cuda") for _ in range(2))
    ctx.mla_q4_decode(capi.mla_config(), q, cache, [n], wuk, wuv, out)
    if finite == 0:
        assert bool(out.isnan().all())
        return
    behind = capi.MlaQ4Cache([cache.codes[0][n - finite:].clone()], [cache.scales[0][n - finite:].clone()],
                             [kr[n - finite:].clone()])
    ctx.mla_q4_decode(capi.mla_config(), q, behind, [finite], wuk, wuv, want)
    # the same scores in both; a weight has three fp16 roundings, the sums' order differs
    most = plain.values(behind.codes[0], behind.scales[0]).abs().sum(1).max() * wuv.double().abs().max()
    assert bool(((out - want).abs() <= 2 * 4 * plain.F16 * most).all())


@pytest.mark.parametrize("n,t,finite", [(300, 300, 200), (300, 300, 236), (3000, 8, 4), (3000, 8, 0), (70, 70, 0)])
def test_prefill_of_infinitely_low_scores(ctx, n, t, finite):
    """Keys that score -inf up to the last `finite` rows: tokens that see no other are NaN, as softmax has it, the
    others as if the sequence began behind them. Whole query tiles and ones cut over the keys (8 tokens after 2992)."""
    import torch

    from pb_b200 import capi

    cfg, bf = capi.mla_config(), torch.bfloat16
    q = _randn((t, 16, NOPE + ROPE), 41)
    q[..., NOPE] = -1.0
    c, k = _randn((n, LAT), 42, 1.0, bf), _randn((n, ROPE), 43, 1.0, bf)
    k[:, 0] = 0.0
    k[:n - finite, 0] = math.inf
    wuk, wuv = _weights()
    out = torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [n])
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache([c], [k]), [n], wuk, wuv, out)
    assert ctx.device_status() == capi.PBMOE_DEV_ERR_F16_RANGE
    rest = min(t, finite)
    assert bool(out[:t - rest].isnan().all())
    if rest:
        # (finite rows before the chunk's first token that sees one: none here)
        want, bound = plain.attend_expanded(q[t - rest:], c[n - finite:], k[n - finite:], wuk, wuv, finite - rest)
        assert bool(((out[t - rest:].double() - want).abs() <= bound).all())
