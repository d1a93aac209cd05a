"""The limits of the latent-attention tests tell a wrong output from a rounded one (CPU): an output of zeros, one with
a tile of rows left out or counted twice, and one that misses a single row are all beyond rms_limit."""

import pytest
import torch

import mla_plain as plain


def _case(n, q_scale):
    g = torch.Generator().manual_seed(n)
    u, s = plain.quantise(torch.randn(n, plain.LAT, generator=g))
    w = [(0.02 * torch.randn(4, d, plain.LAT, generator=g)).bfloat16() for d in (plain.NOPE, plain.V)]
    q = q_scale * torch.randn(4, plain.NOPE + plain.ROPE, generator=g)
    return q, plain.values(plain.pack(u), s), torch.randn(n, plain.ROPE, generator=g).bfloat16(), *w


@pytest.mark.parametrize("n", [200, 1000, 4097, 8000, 30000])
@pytest.mark.parametrize("q_scale", [0.05, 1.0])
def test_wrong_rows_exceed_the_limit(n, q_scale):
    q, lat, kr, wuk, wuv = _case(n, q_scale)
    want = plain.attend_plain(q, lat, kr, wuk, wuv)
    limit = plain.rms_limit(q_scale, bf16_out=True)

    def of(rows):
        return plain.rms(plain.attend_plain(q, lat[rows], kr[rows], wuk, wuv), want)

    rows = torch.arange(n)
    assert plain.rms(torch.zeros_like(want), want) == 1.0 > limit
    for lo in (0, 64 * (n // 128), 64 * ((n - 1) // 64)):  # the first, a middle and the last tile
        tile = rows[lo:lo + 64]
        assert of(torch.cat((rows[:lo], rows[lo + 64:]))) > limit
        assert of(torch.cat((rows, tile))) > limit
    assert of(rows[:-1]) > plain.rms_limit(q_scale)


def test_roundings_stay_below_the_limit():
    """bf16 outputs and weights rounded twice to fp16, as the kernel rounds them, are within it."""
    for n, q_scale in ((200, 1.0), (4097, 1.0), (1000, 0.05)):
        q, lat, kr, wuk, wuv = _case(n, q_scale)
        want = plain.attend_plain(q, lat, kr, wuk, wuv)
        assert plain.rms(want.to(torch.bfloat16), want) <= plain.rms_limit(0.0, True) - plain.rms_limit(0.0)
        s = (torch.einsum("hd,hdc->hc", q[:, :plain.NOPE].double(), wuk.double()).half().double() @ lat.T
             + q[:, plain.NOPE:].double() @ kr.double().T) / (plain.NOPE + plain.ROPE) ** 0.5
        p = torch.exp(s - s.amax(1, keepdim=True))
        p16 = (p.half().float() * 0.73).half().double() / 0.73
        got = torch.einsum("hc,hdc->hd", p16 @ lat / p.sum(1, keepdim=True), wuv.double())
        assert plain.rms(got, want) <= plain.rms_limit(q_scale)
