"""CPU checks of the latent-attention bindings: what they refuse before the C
ABI is reached, the C ABI's refusal of a null context, and the layouts of the
argument structs as a C compiler sees them."""

import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def capi():
    from pb_b200 import build, capi

    build.build()
    return capi


def test_caches_take_cuda_tensors_only(capi):
    import torch

    z = lambda *s, dt=torch.bfloat16: [torch.zeros(*s, dtype=dt)]
    with pytest.raises(ValueError):
        capi.MlaQ4Cache(z(4, 256, dt=torch.uint8), z(4, 8), z(4, 64))
    with pytest.raises(ValueError):
        capi.MlaCache(z(4, 512), z(4, 64))
    with pytest.raises(ValueError):
        capi.MlaQ4Cache([], [], [])
    with pytest.raises(ValueError):
        capi.MlaCache(z(4, 512), [])


def test_host_lengths(capi):
    assert list(capi._host_u32([0, 5, 0xFFFFFFFF], 3, "x")) == [0, 5, 0xFFFFFFFF]
    for bad in ([1, 2], [1, 2, -1], [1, 2, 1 << 32]):
        with pytest.raises(ValueError):
            capi._host_u32(bad, 3, "x")


def test_tensor_checks(capi):
    import torch

    t = torch.zeros(2, 3)
    with pytest.raises(ValueError):  # not on the device
        capi._check(t, "t", (2, 3), (torch.float32,), 0)
    with pytest.raises(TypeError):
        capi._check(t, "t", (2, 3), (torch.bfloat16,), -1)
    with pytest.raises(ValueError):
        capi._check(t, "t", (3, None), (torch.float32,), -1)
    with pytest.raises(ValueError):
        capi._check(t.T, "t", (3, 2), (torch.float32,), -1)
    capi._check(t, "t", (None, 3), (torch.float32,), -1)


def test_null_context(capi):
    lib, cfg, z = capi.load(), capi.mla_config(), C.c_void_p()
    bad = capi.PBMOE_ERR_INVALID_ARGUMENT
    assert lib.pbmoe_mla_q4_append(z, C.byref(cfg), C.byref(capi.MlaQ4AppendArgs()), z) == bad
    assert lib.pbmoe_mla_q4_read(z, C.byref(cfg), 1, z, z, z, z, z, z) == bad
    assert lib.pbmoe_mla_q4_reserve(z, C.byref(cfg), 1) == bad
    assert lib.pbmoe_mla_q4_decode(z, C.byref(cfg), C.byref(capi.MlaQ4Args()), z) == bad
    assert lib.pbmoe_mla_prefill_reserve(z, C.byref(cfg), 1, z, z) == bad
    assert lib.pbmoe_mla_prefill(z, C.byref(cfg), C.byref(capi.MlaPrefillArgs()), z) == bad


def test_struct_layouts(capi, tmp_path):
    structs = {"pbmoe_mla_q4_cache": capi.MlaQ4CacheStruct, "pbmoe_mla_q4_append_args": capi.MlaQ4AppendArgs,
               "pbmoe_mla_q4_args": capi.MlaQ4Args, "pbmoe_mla_prefill_args": capi.MlaPrefillArgs}
    lines = [f'printf("{n} %zu\\n", sizeof({n}));' for n in structs]
    lines += [f'printf("{n}.{f} %zu\\n", offsetof({n}, {f}));' for n, s in structs.items() for f, _ in s._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "pbmoe_cuda.h"\nint main(void) {' + "".join(lines) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for n, s in structs.items():
        assert int(got[n]) == C.sizeof(s)
        for f, _ in s._fields_:
            assert int(got[f"{n}.{f}"]) == getattr(s, f).offset, f"{n}.{f}"


def test_plain_format_round_trip():
    """The quantiser of the tests' plain form: codes within -7..7, values within half a step, zero rows exact."""
    import torch

    import mla_plain as plain

    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, 512, generator=g)
    x[5] = 0
    u, s = plain.quantise(x)
    v = plain.values(plain.pack(u), s)
    assert int(u.min()) >= 1 and int(u.max()) <= 15
    # half a step, and what bf16 takes off the scale (7 steps of 2^-8)
    step = s.double().repeat_interleave(64, 1)
    assert bool(((v - x.double()).abs() <= step * (0.5 + 7 * 2.0**-8)).all())
    assert bool((v[5] == 0).all())
