"""The 4-bit latent cache (pbmoe_mla_q4_append / _read / _decode) against the
plain 64-bit forms of mla_plain.py.

Codes, scales and key rows are compared bit for bit (the format's arithmetic is
f32 division and rounding, the norm's sum is in f64). Decode outputs are held to
the bound of their roundings: with delta the largest error of a score,
  |out - exact| <= (e^(2 delta) - 1 + 3 * 2^-11 + 2^-16) * A + 2^-24 F (+ 2^-8 |out| in bf16),
A = sum_t p_t sum_c |W_UV| |c_t| (3 * 2^-11: p, the scale and their product in
fp16; 2^-16 covers the f32 sums of up to 2^7 additions of terms 16 times the
values they stand for), F = sum_t sum_c |W_UV| |c_t| (fp16 holds a weight below
2^-14 of the largest within 2^-25 of it, twice).
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
    c.rope_reserve(8192, ROPE, 10000.0)
    yield c
    c.close()


def _randn(shape, seed, scale=1.0, dtype=None):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or torch.float32)


def _cache(lens, seed, rows=None):
    """Caches of quantised N(0, 1) rows."""
    import torch

    from pb_b200 import capi

    codes, scales, kr = [], [], []
    for b, n in enumerate(lens):
        r = rows or n
        u, s = plain.quantise(_randn((r, LAT), seed + 10 * b))
        codes.append(plain.pack(u))
        scales.append(s)
        kr.append(_randn((r, ROPE), seed + 10 * b + 1, dtype=torch.bfloat16))
    return capi.MlaQ4Cache(codes, scales, kr)


# ------------------------------------------------------------------ append
def _check_append(ctx, tokens, batch, rows, heads, kv_dtype, q_dtype, out_dtype, norm, seed, in_place=False):
    import torch

    from pb_b200 import capi

    g = torch.Generator()
    g.manual_seed(seed)
    flat = torch.randperm(batch * rows, generator=g)[:tokens] if tokens > batch else \
        torch.arange(batch) * rows + torch.randint(0, rows, (batch,), generator=g)
    seq, pos = (flat // rows).to("cuda", torch.int32), (flat % rows).to("cuda", torch.int32)
    kv = _randn((len(flat), LAT + ROPE), seed, 1.5, kv_dtype)
    w = 1 + 0.2 * _randn((LAT,), seed + 1) if norm else None
    q = _randn((len(flat), heads, NOPE + ROPE), seed + 2, 1.0, q_dtype)
    q0 = q.clone()
    out = q if in_place else torch.full(q.shape, 7.0, dtype=out_dtype, device="cuda")
    cache = capi.MlaQ4Cache.empty(batch, rows)
    for t in cache.codes + cache.scales + cache.k_rope:
        t.view(torch.uint8).fill_(0x5a)
    ctx.mla_q4_append(capi.mla_config(heads=heads), kv, pos, cache, sequences=None if tokens == batch else seq, query=q,
                      query_out=None if in_place else out, latent_norm=w, eps=1e-6)
    assert ctx.device_status() == 0
    lat = kv[:, :LAT].float()
    u, s = plain.quantise(plain.normed(lat, w, 1e-6) if norm else lat)
    li, lp = seq.long().tolist(), pos.long().tolist()
    got_c = torch.stack([cache.codes[b][p] for b, p in zip(li, lp)])
    got_s = torch.stack([cache.scales[b][p] for b, p in zip(li, lp)])
    got_k = torch.stack([cache.k_rope[b][p] for b, p in zip(li, lp)])
    assert torch.equal(got_s.view(torch.int16), s.view(torch.int16))
    assert torch.equal(got_c, plain.pack(u))
    # the table's cos and sin come from two f64 libraries: one f32 step apart at most
    want_k = plain.rope(kv[:, LAT:], pos)
    assert torch.allclose(got_k.float(), want_k, rtol=plain.BF16 * 1.01, atol=1e-6)
    want_q = torch.cat((q0[..., :NOPE].float(), plain.rope(q0[..., NOPE:], pos)), -1)
    tol = plain.BF16 * 1.01 if out.dtype == torch.bfloat16 else 0.0
    assert torch.allclose(out.float(), want_q, rtol=tol, atol=2e-6)
    assert torch.equal(out[..., :NOPE], q0[..., :NOPE].to(out.dtype))
    # every other row as it was
    for b in range(batch):
        keep = torch.ones(rows, dtype=torch.bool)
        keep[[p for i, p in zip(li, lp) if i == b]] = False
        for t in (cache.codes[b], cache.scales[b], cache.k_rope[b]):
            assert bool((t[keep.cuda()].view(torch.uint8) == 0x5a).all())


@pytest.mark.parametrize("tokens,batch,rows,heads", [(1, 1, 1, 16), (1, 1, 4096, 1), (32, 32, 64, 16), (77, 3, 40, 16),
                                                     (300, 5, 513, 128)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(ctx, tokens, batch, rows, heads, norm):
    import torch

    _check_append(ctx, tokens, batch, rows, heads, torch.float32, torch.float32, torch.bfloat16, norm, 3 * tokens + batch)


@pytest.mark.parametrize("kv", ["float32", "bfloat16"])
@pytest.mark.parametrize("q", ["float32", "bfloat16"])
@pytest.mark.parametrize("out", ["float32", "bfloat16"])
def test_append_dtypes(ctx, kv, q, out):
    import torch

    _check_append(ctx, 19, 4, 33, 16, getattr(torch, kv), getattr(torch, q), getattr(torch, out), True, 5)


@pytest.mark.parametrize("q", ["float32", "bfloat16"])
def test_append_in_place(ctx, q):
    import torch

    _check_append(ctx, 19, 4, 33, 16, torch.float32, getattr(torch, q), None, True, 6, in_place=True)


def test_append_no_query_and_nothing(ctx):
    import torch

    from pb_b200 import capi

    cache = capi.MlaQ4Cache.empty(2, 4)
    kv = _randn((2, LAT + ROPE), 1)
    ctx.mla_q4_append(capi.mla_config(), kv, torch.tensor([1, 2], dtype=torch.int32, device="cuda"), cache)
    u, s = plain.quantise(kv[:, :LAT])
    assert torch.equal(cache.codes[0][1], plain.pack(u)[0]) and torch.equal(cache.codes[1][2], plain.pack(u)[1])
    before = cache.codes[0].clone()
    ctx.mla_q4_append(capi.mla_config(), kv[:0], torch.empty(0, dtype=torch.int32, device="cuda"), cache)
    assert torch.equal(cache.codes[0], before)


def test_append_bad_positions_write_nothing(ctx):
    """Rows past a cache or the table, and sequences past the batch, are left out; the others are written."""
    import torch

    from pb_b200 import capi

    cache = capi.MlaQ4Cache([torch.zeros(n, 256, dtype=torch.uint8, device="cuda") for n in (4, 9000)],
                            [torch.zeros(n, 8, dtype=torch.bfloat16, device="cuda") for n in (4, 9000)],
                            [torch.zeros(n, 64, dtype=torch.bfloat16, device="cuda") for n in (4, 9000)])
    i32 = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda").to(torch.int32)
    kv = _randn((6, LAT + ROPE), 2)
    q = _randn((6, 16, NOPE + ROPE), 3)
    q0 = q.clone()
    ctx.mla_q4_append(capi.mla_config(), kv, i32([4, 8192, 3, 5, -1, 8191]), cache, sequences=i32([0, 1, 2, -1, 0, 1]),
                      query=q)
    assert ctx.device_status() == capi.PBMOE_DEV_ERR_POSITION
    assert ctx.device_status() == 0
    assert int(cache.codes[0].sum()) == 0
    assert cache.codes[1].sum(1).nonzero().flatten().tolist() == [8191]
    assert torch.equal(q[:5], q0[:5]) and not torch.equal(q[5], q0[5])


def test_append_extreme_values(ctx):
    """Zero rows, subnormal and huge groups by the format's arithmetic; a non-finite value makes its group NaN."""
    import torch

    from pb_b200 import capi

    kv = _randn((6, LAT + ROPE), 4)
    kv[0, :LAT] = 0
    kv[1, :64] = 0
    kv[2, :64] *= 1e-40
    kv[3, 64:128] *= 1e30
    cache = capi.MlaQ4Cache.empty(6, 2)
    pos = torch.ones(6, dtype=torch.int32, device="cuda")
    ctx.mla_q4_append(capi.mla_config(), kv, pos, cache)
    assert ctx.device_status() == 0
    u, s = plain.quantise(kv[:, :LAT].cpu())  # IEEE arithmetic, subnormals among it
    for b in range(6):
        assert torch.equal(cache.scales[b][1].cpu().view(torch.int16), s[b].view(torch.int16))
        assert torch.equal(cache.codes[b][1].cpu(), plain.pack(u)[b])
    kv[4, 70] = math.nan
    kv[5, 500] = -math.inf
    ctx.mla_q4_append(capi.mla_config(), kv, pos, cache)
    assert ctx.device_status() == capi.PBMOE_DEV_ERR_CACHE_RANGE
    for b, bad in ((4, 1), (5, 7)):
        nan = cache.scales[b][1].isnan()
        assert nan.nonzero().flatten().tolist() == [bad]


@pytest.mark.parametrize("tokens,heads,kv,norm", [(1023, 16, "float32", True), (1024, 16, "float32", True),
                                                  (1201, 3, "bfloat16", False), (2500, 33, "bfloat16", True)])
def test_append_many_tokens(ctx, tokens, heads, kv, norm):
    """Both sides of the number of tokens from which rows are written a warp each, against the format's arithmetic."""
    import torch

    _check_append(ctx, tokens, 3, tokens // 3 + 40, heads, getattr(torch, kv), torch.bfloat16, torch.float32, norm, tokens)


def test_append_many_tokens_as_few(ctx):
    """One call of many tokens writes what calls of few write: bad places, extreme and non-finite values among them."""
    import torch

    from pb_b200 import capi

    n, rows = 1500, 1600
    kv = _randn((n, LAT + ROPE), 44)
    kv[3, :LAT] = 0
    kv[9, 64:128] *= 1e-40
    kv[70, :64] *= 1e30
    kv[801, 70] = math.nan
    kv[1499, 500] = -math.inf
    q = _randn((n, 16, NOPE + ROPE), 45)
    pos = torch.randperm(rows, generator=torch.Generator().manual_seed(1))[:n].to("cuda", torch.int32)
    pos[20], pos[1200] = rows, -1
    seq = torch.zeros(n, dtype=torch.int32, device="cuda")
    seq[77] = 1
    w = 1 + 0.2 * _randn((LAT,), 46)
    many, few = capi.MlaQ4Cache.empty(1, rows), capi.MlaQ4Cache.empty(1, rows)
    q1, q2 = q.clone(), q.clone()
    both = capi.PBMOE_DEV_ERR_POSITION | capi.PBMOE_DEV_ERR_CACHE_RANGE
    ctx.mla_q4_append(capi.mla_config(), kv, pos, many, sequences=seq, query=q1, latent_norm=w)
    assert ctx.device_status() == both
    for i in range(0, n, 300):
        e = slice(i, i + 300)
        ctx.mla_q4_append(capi.mla_config(), kv[e], pos[e], few, sequences=seq[e], query=q2[e], latent_norm=w)
    assert ctx.device_status() == both
    assert torch.equal(q1, q2) and torch.equal(q1[77], q[77])
    for a, b in zip(many.codes + many.scales + many.k_rope, few.codes + few.scales + few.k_rope):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ------------------------------------------------------------------ read back
@pytest.mark.parametrize("begins,counts", [([0], [1]), ([3], [64]), ([0, 5, 0], [65, 0, 200]), ([7, 0], [1, 333]),
                                           (None, [40] * 32)])
def test_read(ctx, begins, counts):
    import torch

    from pb_b200 import capi

    lens = [(begins or [0] * len(counts))[b] + n + 2 for b, n in enumerate(counts)]
    cache = _cache(lens, 21)
    for c in cache.codes:
        c.view(-1)[::5] = 0x0f  # every nibble value, -8 among them
    n = sum(counts)
    pad = torch.full((n + 1, LAT), 3.0, dtype=torch.bfloat16, device="cuda")
    kpad = torch.full((n + 1, ROPE), 3.0, dtype=torch.bfloat16, device="cuda")
    ctx.mla_q4_read(capi.mla_config(), cache, begins, counts, pad[:n], kpad[:n])
    want, wk = [], []
    for b, k in enumerate(counts):
        lo = begins[b] if begins else 0
        want.append(plain.values(cache.codes[b], cache.scales[b])[lo:lo + k])
        wk.append(cache.k_rope[b][lo:lo + k])
    assert torch.equal(pad[:n], torch.cat(want).to(torch.bfloat16))
    assert torch.equal(kpad[:n], torch.cat(wk))
    assert bool((pad[n] == 3).all()) and bool((kpad[n] == 3).all())
    only = torch.empty(n, LAT, dtype=torch.bfloat16, device="cuda")
    ctx.mla_q4_read(capi.mla_config(), cache, begins, counts, only)
    assert torch.equal(only, pad[:n])


# ------------------------------------------------------------------ decode
def _weights(heads, seed, nope=NOPE):
    import torch

    return _randn((heads, nope, LAT), seed, 0.02, torch.bfloat16), _randn((heads, V, LAT), seed + 1, 0.02, torch.bfloat16)


def _bound(mag, flat, delta, out_dtype, want):
    import torch

    b = (torch.expm1(2 * delta) + 3 * plain.F16 + 2.0**-16).view(1, -1, 1) * mag + 2.0**-24 * flat
    return b + (plain.BF16 * want.abs() if out_dtype == torch.bfloat16 else 0) + 1e-30


def _check_decode(ctx, cache, lens, heads=16, q_scale=1.0, q_dtype="float32", out_dtype="float32", nope=NOPE, seed=31,
                  scale=0.0):
    import torch

    from pb_b200 import capi

    wuk, wuv = _weights(heads, seed, nope)
    q = _randn((len(lens), heads, nope + ROPE), seed + 2, q_scale, getattr(torch, q_dtype))
    out = torch.full((len(lens), heads, V), 5.0, dtype=getattr(torch, out_dtype), device="cuda")
    ctx.mla_q4_decode(capi.mla_config(heads=heads, nope=nope, scale=scale), q, cache, lens, wuk, wuv, out)
    for b, n in enumerate(lens):
        lat = plain.values(cache.codes[b][:n], cache.scales[b][:n])
        want, mag, flat, delta = plain.attend(q[b:b + 1], lat, cache.k_rope[b][:n], wuk, wuv,
                                        scale=scale or 1 / math.sqrt(nope + ROPE))
        err = (out[b:b + 1].double() - want).abs()
        lim = _bound(mag, flat, delta, out.dtype, want)
        assert bool((err <= lim).all()), f"seq {b} len {n}: {float((err / lim).max()):.3f} of the bound"
    return out


@pytest.mark.parametrize("lens", [[1], [2], [7], [63], [64], [65], [127], [200], [1000], [3, 130, 64],
                                  [1, 4097, 15, 16, 17, 8000, 511, 512, 513]])
def test_decode(ctx, lens):
    _check_decode(ctx, _cache(lens, 41 + len(lens)), lens)


@pytest.mark.parametrize("heads", [16, 48, 128])
@pytest.mark.parametrize("q_dtype,out_dtype", [("float32", "bfloat16"), ("bfloat16", "float32")])
def test_decode_heads_and_types(ctx, heads, q_dtype, out_dtype):
    lens = [300, 77]
    _check_decode(ctx, _cache(lens, 51), lens, heads, q_dtype=q_dtype, out_dtype=out_dtype)


def test_decode_full_batch(ctx):
    lens = [1 + 37 * b for b in range(32)]
    _check_decode(ctx, _cache(lens, 61), lens)


@pytest.mark.parametrize("q_scale", [0.0, 1e-6, 6.0, 40.0])
def test_decode_score_ranges(ctx, q_scale):
    # 40: a nearly one-hot softmax, its maximum moving from tile to tile
    _check_decode(ctx, _cache([900], 71), [900], q_scale=q_scale)


def test_decode_nope_and_scale(ctx):
    _check_decode(ctx, _cache([90, 5], 72), [90, 5], nope=96, scale=0.25)


def test_decode_rows_behind_the_length_do_not_matter(ctx):
    import torch

    lens = [70, 1]
    cache = _cache(lens, 81, rows=300)
    first = _check_decode(ctx, cache, lens)
    for b, n in enumerate(lens):
        cache.scales[b][n:] = math.nan
        cache.k_rope[b][n:] = math.inf
        cache.codes[b][n:] = 255
    assert torch.equal(_check_decode(ctx, cache, lens), first)


def test_decode_scale_ranges(ctx):
    """Rows of zero, tiny and large scales beside ordinary ones, and groups far apart in one row."""
    lens = [200]
    cache = _cache(lens, 91)
    s = cache.scales[0]
    s[:64] = 0
    s[64:100] *= 2.0**-30
    s[100:110, 3] *= 2.0**12
    _check_decode(ctx, cache, lens, q_scale=0.05)
    s[:] = 0  # a cache that stands for zeros: only the key parts score
    out = _check_decode(ctx, cache, lens)
    assert float(out.abs().max()) == 0.0


def test_decode_nan_scale_stays_in_its_sequence(ctx):
    import torch

    from pb_b200 import capi

    lens = [100, 100, 3]
    cache = _cache(lens, 95)
    clean = _check_decode(ctx, cache, lens)
    cache.scales[1][99, 2] = math.nan
    cache.scales[2][:] = math.nan
    wuk, wuv = _weights(16, 31)
    q = _randn((3, 16, NOPE + ROPE), 33)
    out = torch.empty(3, 16, V, device="cuda")
    ctx.mla_q4_decode(capi.mla_config(), q, cache, lens, wuk, wuv, out)
    assert torch.equal(out[0], clean[0])
    assert bool(out[1].isnan().all()) and bool(out[2].isnan().all())


def test_decode_nan_query_stays_in_its_head(ctx):
    import torch

    from pb_b200 import capi

    lens = [130, 5]
    cache = _cache(lens, 97)
    clean = _check_decode(ctx, cache, lens)
    wuk, wuv = _weights(16, 31)
    q = _randn((2, 16, NOPE + ROPE), 33)
    q[0, 3, 7] = math.nan
    q[1, 9, NOPE + 1] = math.inf
    out = torch.empty(2, 16, V, device="cuda")
    ctx.mla_q4_decode(capi.mla_config(), q, cache, lens, wuk, wuv, out)
    bad = torch.zeros(2, 16, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[1, 9] = True
    assert torch.equal(out[~bad], clean[~bad]) and bool(out[bad].isnan().all())


def test_rows_of_weight_zero_before_low_scores(ctx):
    """Rows that score -inf (a whole tile and more), then scores far below zero: as if the sequence began behind them."""
    import torch

    from pb_b200 import capi

    n, lost = 200, 64
    cache = _cache([n], 99)
    q = _randn((1, 16, NOPE + ROPE), 34)
    # times the scale in base 2: -1.001, which is not a bf16, so neither half of it is 0
    q[..., NOPE] = -1.001 * math.sqrt(NOPE + ROPE) * math.log(2)
    q[..., NOPE + 1] = -100.0
    kr = cache.k_rope[0]
    kr[:, 0], kr[:, 1] = 0.0, 1000.0
    kr[:lost, 0] = math.inf
    behind = capi.MlaQ4Cache([cache.codes[0][lost:]], [cache.scales[0][lost:]], [kr[lost:]])
    wuk, wuv = _weights(16, 31)
    out, want = torch.empty(1, 16, V, device="cuda"), torch.empty(1, 16, V, device="cuda")
    ctx.mla_q4_decode(capi.mla_config(), q, cache, [n], wuk, wuv, out)
    ctx.mla_q4_decode(capi.mla_config(), q, behind, [n - lost], wuk, wuv, want)
    # the same scores in both; a weight has three fp16 roundings, the sums' order differs
    most = plain.values(cache.codes[0], cache.scales[0]).abs().sum(1).max() * wuv.double().abs().max()
    assert bool(out.isfinite().all()) and bool(((out - want).abs() <= 2 * 4 * plain.F16 * most).all())


def test_same_cache_for_several_sequences(ctx):
    """Sequences that share a buffer (a common prefix at different lengths) read it side by side."""
    import torch

    from pb_b200 import capi

    one = _cache([500], 98)
    lens = [500, 17, 64, 333]
    cache = capi.MlaQ4Cache(one.codes * 4, one.scales * 4, one.k_rope * 4)
    _check_decode(ctx, cache, lens)


def test_decode_offsets_past_32_bits(ctx):
    """A cache of over 4 GiB of codes: the attended rows at its end are the only ones that stand for anything."""
    import torch

    from pb_b200 import capi

    n = (1 << 24) + 100
    codes = torch.full((n, 256), 0x88, dtype=torch.uint8, device="cuda")  # q = 0
    scales = torch.ones(n, 8, dtype=torch.bfloat16, device="cuda")
    kr = torch.zeros(n, 64, dtype=torch.bfloat16, device="cuda")
    u, s = plain.quantise(_randn((90, LAT), 7))
    codes[n - 90:], scales[n - 90:] = plain.pack(u), s
    kr[n - 90:] = 4.0
    cache = capi.MlaQ4Cache([codes], [scales], [kr])
    got = torch.empty(90, LAT, dtype=torch.bfloat16, device="cuda")
    ctx.mla_q4_read(capi.mla_config(), cache, [n - 90], [90], got)
    assert torch.equal(got, plain.values(plain.pack(u), s).to(torch.bfloat16))
    wuk, wuv = _weights(16, 8)
    q = torch.full((1, 16, NOPE + ROPE), 0.0, device="cuda")
    q[..., NOPE:] = 1.2  # the last rows score 64 * 4.8 / sqrt(192) = 22.2, the others 0
    out = torch.empty(1, 16, V, device="cuda")
    ctx.mla_q4_decode(capi.mla_config(), q, cache, [n], wuk, wuv, out)
    e = math.exp(64 * 1.2 * 4 / math.sqrt(192))  # q 1.2 in f32
    lat = plain.values(plain.pack(u), s)
    p = e / (e * 90 + (n - 90))
    ctxv = p * lat.sum(0)
    want = torch.einsum("hdc,c->hd", wuv.double(), ctxv)
    mag = torch.einsum("hdc,c->hd", wuv.double().abs(), p * lat.abs().sum(0))
    # score error: f32 sums and Q' hi + lo (2^-16 each way) of 22.2; sum of 2^24 ones in f32 partials
    assert bool(((out[0].double() - want).abs() <= (22.2 * 2 * 2.0**-15 + 3 * plain.F16 + 2.0**-12) * mag).all())


def test_append_then_decode(ctx):
    """Prompt rows and then one token a sequence, as a decode step runs them, on another stream than the default."""
    import torch

    from pb_b200 import capi

    cfg, lens = capi.mla_config(), [33, 150]
    cache = capi.MlaQ4Cache.empty(2, 256)
    wuk, wuv = _weights(16, 3)
    w = 1 + 0.1 * _randn((LAT,), 4)
    seq = torch.cat([torch.full((n,), b) for b, n in enumerate(lens)]).to("cuda", torch.int32)
    pos = torch.cat([torch.arange(n) for n in lens]).to("cuda", torch.int32)
    kv, kv1 = _randn((sum(lens), LAT + ROPE), 5), _randn((2, LAT + ROPE), 6)
    q1, out = _randn((2, 16, NOPE + ROPE), 7), torch.empty(2, 16, V, device="cuda")
    last = torch.tensor(lens, dtype=torch.int32, device="cuda")
    rotated = torch.empty_like(q1)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    ctx.mla_q4_append(cfg, kv, pos, cache, sequences=seq, latent_norm=w, stream=st)
    ctx.mla_q4_append(cfg, kv1, last, cache, query=q1, query_out=rotated, latent_norm=w, stream=st)
    ctx.mla_q4_decode(cfg, rotated, cache, [n + 1 for n in lens], wuk, wuv, out, stream=st)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        rows = torch.cat((kv[seq == b], kv1[b:b + 1]))
        u, s = plain.quantise(plain.normed(rows[:, :LAT], w, 1e-6))
        kr = plain.rope(rows[:, LAT:], torch.arange(n + 1, device="cuda")).to(torch.bfloat16)
        qr = torch.cat((q1[b:b + 1, :, :NOPE], plain.rope(q1[b:b + 1, :, NOPE:], last[b:b + 1])), -1)
        want, mag, flat, delta = plain.attend(qr, plain.values(plain.pack(u), s), kr, wuk, wuv)
        # key rows one bf16 step apart where cos/sin differ in the last place: rare, within 2^-11 on every score
        lim = _bound(mag, flat, delta + 1e-4, torch.float32, want)
        assert bool(((out[b:b + 1].double() - want).abs() <= lim).all())


def test_graph_replay_and_two_contexts(ctx):
    """A captured append + decode replayed on new inputs gives what eager calls give; a second context's calls on
    another stream do not disturb it."""
    import torch

    from pb_b200 import capi

    cfg, lens = capi.mla_config(), [400, 90]
    other = capi.Context(0)
    other.mla_q4_reserve(cfg, 2)
    cache = _cache(lens, 13)
    wuk, wuv = _weights(16, 14)
    kv = _randn((2, LAT + ROPE), 15)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device="cuda")
    q, rot = _randn((2, 16, NOPE + ROPE), 16), torch.empty(2, 16, NOPE + ROPE, device="cuda")
    out, want, out2 = (torch.empty(2, 16, V, device="cuda") for _ in range(3))

    def step(o):
        ctx.mla_q4_append(cfg, kv, pos, cache, query=q, query_out=rot)
        ctx.mla_q4_decode(cfg, rot, cache, lens, wuk, wuv, o)

    step(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(out)
    side = torch.cuda.Stream()
    for seed in range(3):
        kv.copy_(_randn((2, LAT + ROPE), 100 + seed))
        q.copy_(_randn((2, 16, NOPE + ROPE), 200 + seed))
        out.zero_()
        torch.cuda.synchronize()
        still = _cache(lens, 300)
        other.mla_q4_decode(cfg, q, still, lens, wuk, wuv, out2, stream=side)
        graph.replay()
        torch.cuda.synchronize()
        step(want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    other.close()


# ------------------------------------------------------------------ refusals
def test_refusals(ctx):
    import torch

    from pb_b200 import capi

    cfg = capi.mla_config()
    cache = _cache([8, 8], 1)
    wuk, wuv = _weights(16, 1)
    q, out = _randn((2, 16, NOPE + ROPE), 1), torch.full((2, 16, V), 9.0, device="cuda")

    def code(fn, *a, **k):
        with pytest.raises(capi.PbmoeError) as e:
            fn(*a, **k)
        return e.value.code

    INV, UNS, WS = capi.PBMOE_ERR_INVALID_ARGUMENT, capi.PBMOE_ERR_UNSUPPORTED, capi.PBMOE_ERR_NO_WORKSPACE
    assert code(ctx.mla_q4_decode, cfg, q, cache, [0, 8], wuk, wuv, out) == INV
    assert code(ctx.mla_q4_decode, cfg, q, cache, [8, 9], wuk, wuv, out) == INV
    h8 = capi.mla_config(heads=8)
    assert code(ctx.mla_q4_decode, h8, q[:, :8].contiguous(), cache, [8, 8], wuk[:8], wuv[:8], out[:, :8].contiguous()) == UNS
    assert code(ctx.mla_q4_reserve, capi.mla_config(heads=144), 1) == UNS
    assert code(ctx.mla_q4_reserve, cfg, 33) == INV
    assert code(ctx.mla_q4_reserve, capi.mla_config(scale=math.inf), 1) == INV
    fresh = capi.Context(0)
    assert code(fresh.mla_q4_decode, cfg, q, cache, [8, 8], wuk, wuv, out) == WS
    kv, pos = _randn((2, LAT + ROPE), 1), torch.zeros(2, dtype=torch.int32, device="cuda")
    assert code(fresh.mla_q4_append, cfg, kv, pos, cache) == WS  # no RoPE table
    fresh.close()
    kv3, pos3 = _randn((3, LAT + ROPE), 1), torch.zeros(3, dtype=torch.int32, device="cuda")
    assert code(ctx.mla_q4_append, cfg, kv3, pos3, cache) == INV  # three tokens of two sequences
    assert code(ctx.mla_q4_append, cfg, kv, pos, cache, latent_norm=torch.ones(LAT, device="cuda"), eps=-1.0) == INV
    assert code(ctx.mla_q4_append, cfg, kv, pos, cache, query_out=q) == INV
    rows = torch.empty(16, LAT, dtype=torch.bfloat16, device="cuda")
    assert code(ctx.mla_q4_read, cfg, cache, [1, 0], [8, 8], rows) == INV
    with pytest.raises(ValueError):
        ctx.mla_q4_read(cfg, cache, None, [8, 8], rows[:15])
    with pytest.raises(ValueError):
        ctx.mla_q4_decode(cfg, q.transpose(0, 1), cache, [8, 8], wuk, wuv, out)
    with pytest.raises(TypeError):
        ctx.mla_q4_decode(cfg, q.half(), cache, [8, 8], wuk, wuv, out)
    with pytest.raises(ValueError):
        ctx.mla_q4_decode(cfg, q.cpu(), cache, [8, 8], wuk, wuv, out)
    with pytest.raises(ValueError):
        ctx.mla_q4_decode(cfg, q, cache, [8], wuk, wuv, out)
    torch.cuda.synchronize()
    assert bool((out == 9).all())
    # misaligned buffers, straight through the C ABI
    import ctypes as C

    bad = capi.MlaQ4CacheStruct(cache.codes[0].data_ptr() + 8, cache.scales[0].data_ptr(), cache.k_rope[0].data_ptr(), 4)
    lens = (C.c_uint32 * 1)(4)
    a = capi.MlaQ4Args(1, C.addressof(lens), q.data_ptr(), 0, C.addressof(bad), wuk.data_ptr(), wuv.data_ptr(),
                       out.data_ptr(), 0)
    assert ctx.lib.pbmoe_mla_q4_decode(ctx.h, C.byref(cfg), C.byref(a), None) == INV
    assert "16-byte" in ctx.last_error()
    big = capi.MlaQ4CacheStruct(cache.codes[0].data_ptr(), cache.scales[0].data_ptr(), cache.k_rope[0].data_ptr(), 1 << 31)
    a.caches = C.addressof(big)
    assert ctx.lib.pbmoe_mla_q4_decode(ctx.h, C.byref(cfg), C.byref(a), None) == UNS
    assert ctx.lib.pbmoe_mla_q4_decode(None, C.byref(cfg), C.byref(a), None) == INV
    assert ctx.lib.pbmoe_mla_q4_decode(ctx.h, C.byref(cfg), None, None) == INV
