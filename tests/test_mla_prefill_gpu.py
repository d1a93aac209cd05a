"""pbmoe_mla_prefill (causal latent attention of prompt chunks, expanded form)
against the plain 64-bit form of mla_plain.py, element by element within the
bound of its fp16 roundings (attend_expanded); bf16 outputs add 2^-8 |out|."""

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
    yield c
    c.close()


def _randn(shape, seed, scale=1.0, dtype=None):
    import torch

    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or torch.float32)


def _inputs(q_lens, lens, heads, seed, q_scale, q_dtype):
    import torch

    bf = torch.bfloat16
    c = [_randn((n, LAT), seed + 10 * b, 1.0, bf) for b, n in enumerate(lens)]
    k = [_randn((n, ROPE), seed + 10 * b + 1, 1.0, bf) for b, n in enumerate(lens)]
    return (_randn((sum(q_lens), heads, NOPE + ROPE), seed + 2, q_scale, q_dtype), c, k,
            _randn((heads, NOPE, LAT), seed + 3, 0.02, bf), _randn((heads, V, LAT), seed + 4, 0.02, bf))


def _within(got, want, bound, q_scale=1.0):
    """Every element within its bound, and the whole within what random roundings add up to. A score is a sum of terms
    with two rounded factors, each off by 2^-11 / sqrt(3) at random: its error is 2^-11 sqrt(2/3) of the scores' own
    deviation, which these inputs make 0.69 q_scale (sqrt((128 * 0.205 + 64) / 192)): below 2^-11 q_scale. An output
    moves by at most that share of itself, beside the roundings of p, V and the output."""
    import torch

    lim = bound + (plain.BF16 * want.abs() if got.dtype == torch.bfloat16 else 0)
    err = (got.double() - want).abs()
    assert bool((err <= lim).all()), f"{float((err / lim).max()):.3f} of the bound"
    rms = float(err.norm() / want.norm().clamp_min(1e-30))
    assert rms <= (3e-3 if got.dtype == torch.bfloat16 else 1e-3) + plain.F16 * q_scale or float(want.norm()) == 0, rms


def _run(ctx, q_lens, lens, heads=16, q_scale=1.0, q_dtype="float32", out_dtype="float32", seed=3, scale=0.0, check=True):
    import torch

    from pb_b200 import capi

    cfg = capi.mla_config(heads=heads, scale=scale)
    q, c, k, wuk, wuv = _inputs(q_lens, lens, heads, seed, q_scale, getattr(torch, q_dtype))
    out = torch.full((sum(q_lens) + 1, heads, V), 7.0, dtype=getattr(torch, out_dtype), device="cuda")
    ctx.mla_prefill_reserve(cfg, q_lens, lens)
    ctx.mla_prefill(cfg, q, q_lens, capi.MlaCache(c, k), lens, wuk, wuv, out[:-1])
    assert ctx.device_status() == 0
    assert bool((out[-1] == 7).all())
    at = 0
    for b, (t, n) in enumerate(zip(q_lens, lens)):
        if t and check:
            want, bound = plain.attend_expanded(q[at:at + t], c[b], k[b], wuk, wuv, n - t, scale)
            _within(out[at:at + t], want, bound, q_scale)
        at += t
    return out[:-1]


@pytest.mark.parametrize("t", [1, 2, 127, 128, 129, 255, 256, 257, 500])
def test_prompt(ctx, t):
    _run(ctx, [t], [t])


@pytest.mark.parametrize("t,n", [(1, 2), (1, 128), (1, 129), (1, 1000), (3, 130), (61, 4096), (128, 256), (130, 385),
                                 (300, 1333)])
def test_chunk_after_context(ctx, t, n):
    _run(ctx, [t], [n], seed=t + n)


@pytest.mark.parametrize("q_lens,lens", [([5, 200], [5, 333]), ([0, 3, 0, 700, 1], [50, 3, 0, 900, 640]),
                                         ([1] * 32, [1 + 9 * b for b in range(32)])])
def test_ragged_batch(ctx, q_lens, lens):
    _run(ctx, q_lens, lens)


@pytest.mark.parametrize("heads", [1, 3, 16, 128])
@pytest.mark.parametrize("q_dtype,out_dtype", [("float32", "bfloat16"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")])
def test_heads_and_types(ctx, heads, q_dtype, out_dtype):
    _run(ctx, [140, 9], [300, 9], heads, q_dtype=q_dtype, out_dtype=out_dtype)


@pytest.mark.parametrize("q_scale", [0.0, 1e-4, 8.0, 60.0])
def test_score_ranges(ctx, q_scale):
    _run(ctx, [300], [700], q_scale=q_scale)


def test_softmax_scale(ctx):
    _run(ctx, [90], [90], scale=0.3)


def test_rising_scores_move_the_maximum(ctx):
    """Keys that grow along the cache: every tile exceeds the running maximum by more than 2^8."""
    import torch

    from pb_b200 import capi

    cfg, n, t = capi.mla_config(), 1024, 200
    q, c, k, wuk, wuv = _inputs([t], [n], 16, 9, 1.0, torch.float32)
    q[..., NOPE:] = 1.0
    k[0][:] = (torch.arange(n, device="cuda") / 64).unsqueeze(1).to(torch.bfloat16)
    out = torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [n])
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [n], wuk, wuv, out)
    want, bound = plain.attend_expanded(q, c[0], k[0], wuk, wuv, n - t)
    _within(out, want, bound)


def test_long_prompt(ctx):
    _run(ctx, [2500], [4100], heads=2)


def test_more_query_tiles_than_a_work_list(ctx):
    """Over 512 query tiles in one call (131072 rows): single rows of it against the plain form."""
    import torch

    from pb_b200 import capi

    cfg, q_lens, lens = capi.mla_config(heads=1), [70001, 300, 69999], [70001, 900, 70100]
    q, c, k, wuk, wuv = _inputs(q_lens, lens, 1, 17, 1.0, torch.bfloat16)
    out = torch.empty(sum(q_lens), 1, V, dtype=torch.bfloat16, device="cuda")
    ctx.mla_prefill_reserve(cfg, q_lens, lens)
    ctx.mla_prefill(cfg, q, q_lens, capi.MlaCache(c, k), lens, wuk, wuv, out)
    assert ctx.device_status() == 0
    first = 0
    for b, (t, n) in enumerate(zip(q_lens, lens)):
        for i in (0, t // 2 + 1, t - 1):
            seen = n - t + i + 1
            want, bound = plain.attend_expanded(q[first + i:first + i + 1], c[b][:seen], k[b][:seen], wuk, wuv, seen - 1)
            err = (out[first + i:first + i + 1].double() - want).abs()
            assert bool((err <= bound + plain.BF16 * want.abs()).all())
        first += t


def test_nan_query_stays_in_its_row(ctx):
    import torch

    from pb_b200 import capi

    cfg, t, n = capi.mla_config(), 140, 300
    q, c, k, wuk, wuv = _inputs([t], [n], 16, 19, 1.0, torch.float32)
    out, clean = torch.empty(t, 16, V, device="cuda"), torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [n])
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [n], wuk, wuv, clean)
    bad = torch.zeros(t, 16, dtype=torch.bool, device="cuda")
    for row, head in ((0, 0), (77, 5), (139, 15)):
        q[row, head, 3] = math.nan
        bad[row, head] = True
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [n], wuk, wuv, out)
    assert ctx.device_status() == capi.PBMOE_DEV_ERR_F16_RANGE
    assert torch.equal(out[~bad], clean[~bad]) and bool(out[bad].isnan().all())


def test_rows_that_are_not_seen_do_not_matter(ctx):
    """NaN and infinity in a later row of the chunk: earlier tokens keep their outputs, later ones follow the formula
    (an infinite key part scores +inf or -inf by the query's sign: NaN, or a weight of 0)."""
    import torch

    from pb_b200 import capi

    cfg, t = capi.mla_config(), 300
    q, c, k, wuk, wuv = _inputs([t], [t], 16, 21, 1.0, torch.float32)
    out, clean = torch.empty(t, 16, V, device="cuda"), torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [t])
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [t], wuk, wuv, clean)
    for bad, tensor in ((math.nan, c[0]), (math.inf, k[0])):
        keep = tensor[200].clone()
        tensor[200, 7] = bad
        ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [t], wuk, wuv, out)
        assert ctx.device_status() == capi.PBMOE_DEV_ERR_F16_RANGE
        assert torch.equal(out[:200], clean[:200])
        hit = q[200:, :, NOPE + 7] > 0 if tensor is k[0] else torch.ones(t - 200, 16, dtype=torch.bool, device="cuda")
        assert torch.equal(out[200:].isnan(), hit.unsqueeze(-1).expand(-1, -1, V))
        tensor[200] = keep
    q[100, 3, 0] = 1e6
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [t], wuk, wuv, out)
    assert ctx.device_status() == capi.PBMOE_DEV_ERR_F16_RANGE


@pytest.mark.parametrize("lost,n,t", [(64, 300, 150), (1024, 3000, 8)])
def test_rows_of_weight_zero_before_low_scores(ctx, lost, n, t):
    """Whole key tiles that score -inf, then scores far below zero: as if the sequence began behind them."""
    import torch

    from pb_b200 import capi

    cfg = capi.mla_config()
    q, c, k, wuk, wuv = _inputs([t], [n], 16, 23, 1.0, torch.float32)
    q[..., NOPE], q[..., NOPE + 1] = -1.0, -100.0
    k[0][:, 0], k[0][:, 1] = 0.0, 1000.0  # -7000 to every score
    k[0][:lost, 0] = math.inf
    out, want = torch.empty(t, 16, V, device="cuda"), torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [n])
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [n], wuk, wuv, out)
    assert ctx.device_status() == capi.PBMOE_DEV_ERR_F16_RANGE
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache([c[0][lost:]], [k[0][lost:]]), [n - lost], wuk, wuv, want)
    # the same scores in both; the weights' roundings (fp16, and the exponential's 2^-13) may differ, the sums' order too
    most = (c[0].double() @ wuv.double().transpose(1, 2)).abs().amax()
    assert bool(((out - want).abs() <= 2 * (plain.F16 + 2.0**-13 + 2.0**-16) * most).all())


def test_cache_rows_behind_the_sequence_are_not_read(ctx):
    import torch

    from pb_b200 import capi

    cfg, t, n = capi.mla_config(), 40, 150
    q, c, k, wuk, wuv = _inputs([t], [300], 16, 23, 1.0, torch.float32)
    q = q[:t].contiguous()
    out, clean = torch.empty(t, 16, V, device="cuda"), torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [n])
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [n], wuk, wuv, clean)
    c[0][n:] = math.nan
    k[0][n:] = math.nan
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [n], wuk, wuv, out)
    assert ctx.device_status() == 0
    assert torch.equal(out, clean)


def test_same_as_decode_and_from_the_4bit_cache(ctx):
    """A chunked prompt as it is served: rows appended to the 4-bit cache, read back, attended by the chunk; its last
    token equals a decode step over the same cache."""
    import torch

    from pb_b200 import capi

    cfg, n, t = capi.mla_config(), 333, 77
    ctx.rope_reserve(4096, ROPE, 10000.0)
    ctx.mla_q4_reserve(cfg, 1)
    ctx.mla_prefill_reserve(cfg, [t], [n])
    q, _, _, wuk, wuv = _inputs([n], [1], 16, 31, 1.0, torch.float32)
    kv, w = _randn((n, LAT + ROPE), 32), 1 + 0.1 * _randn((LAT,), 33)
    cache = capi.MlaQ4Cache.empty(1, 400)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    rot = torch.empty_like(q)
    ctx.mla_q4_append(cfg, kv, pos, cache, sequences=seq, query=q, query_out=rot, latent_norm=w)
    c = torch.empty(n, LAT, dtype=torch.bfloat16, device="cuda")
    k = torch.empty(n, ROPE, dtype=torch.bfloat16, device="cuda")
    ctx.mla_q4_read(cfg, cache, None, [n], c, k)
    out = torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill(cfg, rot[n - t:], [t], capi.MlaCache([c], [k]), [n], wuk, wuv, out)
    one = torch.empty(1, 16, V, device="cuda")
    ctx.mla_q4_decode(cfg, rot[n - 1:], cache, [n], wuk, wuv, one)
    torch.cuda.synchronize()
    want, bound = plain.attend_expanded(rot[n - t:], c, k, wuk, wuv, n - t)
    _within(out, want, bound)
    # the decode reads q s itself, the chunk its bf16: 2^-8 of every latent value more
    rms = float((one[0] - out[-1]).norm() / out[-1].norm())
    assert rms <= plain.BF16 + 2e-3, rms


@pytest.mark.parametrize("t,rows", [(70, 200), (1100, 1100)])
def test_calls_back_to_back(ctx, t, rows):
    """Append, read back, prefill and decode over shared buffers, again and again without a wait: each launch starts
    before the one ahead of it has ended, and what it reads has to be that one's."""
    import torch

    from pb_b200 import capi

    cfg, n = capi.mla_config(), 6
    ctx.rope_reserve(4096, 64)
    ctx.mla_q4_reserve(cfg, 1)
    ctx.mla_prefill_reserve(cfg, [t], [rows])
    g = torch.Generator(device="cuda").manual_seed(t)
    kv = torch.randn(n, rows, 576, device="cuda", generator=g)
    q = torch.randn(n, rows, 16, 192, device="cuda", generator=g)
    wuk, wuv = (0.05 * torch.randn(16, 128, 512, device="cuda", generator=g).bfloat16() for _ in range(2))
    cache, pos = capi.MlaQ4Cache.empty(1, rows), torch.arange(rows, dtype=torch.int32, device="cuda")
    seq, rot = torch.zeros_like(pos), torch.empty(rows, 16, 192, dtype=torch.bfloat16, device="cuda")
    c, k = torch.empty(rows, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(rows, 64, dtype=torch.bfloat16, device="cuda")
    kept = capi.MlaCache([c], [k])

    def run(wait):
        out, one = torch.zeros(n, t, 16, V, device="cuda"), torch.zeros(n, 1, 16, V, device="cuda")
        for i in range(n):
            for call in (lambda: ctx.mla_q4_append(cfg, kv[i], pos, cache, sequences=seq, query=q[i], query_out=rot),
                         lambda: ctx.mla_q4_read(cfg, cache, None, [rows], c, k),
                         lambda: ctx.mla_prefill(cfg, rot[rows - t:], [t], kept, [rows], wuk, wuv, out[i]),
                         lambda: ctx.mla_q4_decode(cfg, rot[rows - 1:], cache, [rows], wuk, wuv, one[i])):
                call()
                if wait:
                    torch.cuda.synchronize()
        return out, one

    want = run(True)
    assert ctx.device_status() == 0 and bool(want[0].any(-1).all())
    for _ in range(3):
        got = run(False)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_graph_replay_on_another_stream(ctx):
    import torch

    from pb_b200 import capi

    cfg, t, n = capi.mla_config(), 200, 300
    q, c, k, wuk, wuv = _inputs([t], [n], 16, 41, 1.0, torch.float32)
    kept = capi.MlaCache(c, k)
    out, want = torch.empty(t, 16, V, device="cuda"), torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [n])
    ctx.mla_prefill(cfg, q, [t], kept, [n], wuk, wuv, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.mla_prefill(cfg, q, [t], kept, [n], wuk, wuv, out)
    for seed in range(3):
        q.copy_(_randn(q.shape, 50 + seed))
        c[0].copy_(_randn(c[0].shape, 60 + seed))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        ctx.mla_prefill(cfg, q, [t], kept, [n], wuk, wuv, want, stream=st)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_refusals(ctx):
    import torch

    from pb_b200 import capi

    cfg = capi.mla_config()
    q, c, k, wuk, wuv = _inputs([4], [8], 16, 1, 1.0, torch.float32)
    kept = capi.MlaCache(c, k)
    out = torch.full((4, 16, V), 9.0, device="cuda")
    INV, UNS, WS = capi.PBMOE_ERR_INVALID_ARGUMENT, capi.PBMOE_ERR_UNSUPPORTED, capi.PBMOE_ERR_NO_WORKSPACE

    def code(fn, *a):
        with pytest.raises(capi.PbmoeError) as e:
            fn(*a)
        return e.value.code

    fresh = capi.Context(0)
    assert code(fresh.mla_prefill, cfg, q, [4], kept, [8], wuk, wuv, out) == WS
    fresh.close()
    ctx.mla_prefill_reserve(cfg, [4], [8])
    assert code(ctx.mla_prefill, cfg, q, [4], kept, [3], wuk, wuv, out) == INV
    assert code(ctx.mla_prefill_reserve, capi.mla_config(heads=129), [1], [1]) == UNS
    assert code(ctx.mla_prefill_reserve, capi.mla_config(nope=64), [1], [1]) == UNS
    assert code(ctx.mla_prefill_reserve, cfg, [1] * 33, [1] * 33) == INV
    assert code(ctx.mla_prefill_reserve, cfg, [1 << 24], [1 << 24]) == UNS
    assert code(ctx.mla_prefill_reserve, cfg, [2], [1]) == INV
    with pytest.raises(ValueError):
        ctx.mla_prefill(cfg, q, [4], kept, [9], wuk, wuv, out)
    with pytest.raises(ValueError):
        ctx.mla_prefill(cfg, q, [3], kept, [8], wuk, wuv, out)
    with pytest.raises(TypeError):
        ctx.mla_prefill(cfg, q.half(), [4], kept, [8], wuk, wuv, out)
    with pytest.raises(ValueError):
        ctx.mla_prefill(cfg, q, [4], kept, [8], wuk, wuv, out.cpu())
    ctx.mla_prefill(cfg, q[:0], [0], kept, [8], wuk, wuv, out[:0])  # nothing to do
    torch.cuda.synchronize()
    assert bool((out == 9).all())


@pytest.mark.parametrize("heads,t,n", [(1, 1, 1001), (1, 500, 1500), (1, 1024, 1024), (4, 256, 1256), (4, 4096, 4096),
                                       (16, 500, 1500), (32, 1, 1001), (32, 256, 5000)])
def test_cut_query_tiles(ctx, heads, t, n):
    """Shapes whose query tiles are cut over the keys and joined, in 3 to 6 parts, some parts empty for early rows."""
    _run(ctx, [t], [n], heads, seed=t + n + heads)


@pytest.mark.parametrize("factor", [2.0**-6, 2.0**-12, 2.0**-18])
def test_small_latents(ctx, factor):
    """Keys and values below fp16's normal range: within 2^-25 a value, which the bound counts."""
    import torch

    from pb_b200 import capi

    cfg, t, n = capi.mla_config(), 150, 400
    q, c, k, wuk, wuv = _inputs([t], [n], 16, 61, 1.0, torch.float32)
    c[0].mul_(factor)
    out = torch.empty(t, 16, V, device="cuda")
    ctx.mla_prefill_reserve(cfg, [t], [n])
    ctx.mla_prefill(cfg, q, [t], capi.MlaCache(c, k), [n], wuk, wuv, out)
    assert ctx.device_status() == 0
    want, bound = plain.attend_expanded(q, c[0], k[0], wuk, wuv, n - t)
    assert bool(((out.double() - want).abs() <= bound).all())
