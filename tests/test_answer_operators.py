"""The kernels for rotation on the way into the cache, adapters and log probabilities without a GPU: every form compiles, bad parameters and
operands are refused."""
import pytest
import torch

from kernelcodegen_amd import _lib, ops, runtime as R
from test_decode_step import WRITE, cache

APPEND = dict(WRITE, R=64, PAIRS=0, HQ=4, QN=1, XQT=512, XQH=128)
ADAPT = dict(N=1000, K=4096, RANK=16, F16=0, Y_F32=0, XT=4096, YT=1000, ZT=1000, ALIGN=1)
LOGPROBS = dict(V=32000, F16=2, TOP=5, STRIDE=32000)
GOOD = [("cache_append", dict(cache(d), **{**APPEND, "R": r, "F16": f16, "WIN": win, "PAIRS": pairs}), 14)
        for d, r, f16, win, pairs in ((128, 128, 2, 1, 0), (96, 96, 0, 16, 1), (256, 32, 1, 4, 0), (32, 16, 2, 16, 1), (224, 224, 0, 1, 0), (160, 80, 1, 16, 0))]
GOOD += [(family, dict(ADAPT, **more), 10 if family.endswith("up") else 7) for family in ("adapters_down", "adapters_up")
         for more in (dict(), dict(RANK=8, F16=1, Y_F32=1, SCALES=1, MANY=1, KS=8), dict(RANK=256, K=264, UT=4, MANY=1), dict(RANK=64, TS=4, UT=4, KS=2), dict(RANK=128, TS=2, UT=2, Y_F32=1, F16=1), dict(RANK=24, N=77, YT=77, ZT=77, ALIGN=0, INPLACE=1), dict(N=4))]
GOOD += [("token_logprobs", dict(LOGPROBS, **more), 6) for more in (dict(), dict(TOP=0, F16=1), dict(F16=0, TOP=32), dict(V=1, TOP=1, STRIDE=0), dict(V=1 << 19, F16=0, STRIDE=1 << 19), dict(V=50021, STRIDE=50021, SHIFT=1))]
GOOD += [("token_logprobs", dict(LOGPROBS, SPLIT=1, THREADS=256), 3), ("logprobs_join", dict(LOGPROBS, THREADS=256), 8)]


@pytest.mark.parametrize("family,params,nargs", GOOD)
def test_every_form_compiles_for_gfx950(family, params, nargs):
    text, info = R.emit_kernel(family, "kernel0", **params)
    assert info["name"] == "kernel0" and info["num_args"] == nargs and info["workspace_bytes"] == 0
    assert R.compile_to_code(R.prelude() + text)[:4] == b"\x7fELF"


@pytest.mark.parametrize("family,params", [
    ("cache_append", dict(cache(64), **{**APPEND, "R": 24})), ("cache_append", dict(cache(32), **APPEND)), ("cache_append", dict(cache(64), **{**APPEND, "R": 0})),
    ("cache_append", dict(cache(64), **{**APPEND, "HQ": 0})), ("cache_append", dict(cache(64), **{**APPEND, "QN": 9})), ("cache_append", dict(cache(64), **{**APPEND, "XQT": 4})),
    ("cache_append", dict(cache(64), **WRITE)), ("cache_append", dict(cache(48), **APPEND)),
    ("adapters_up", dict(ADAPT, RANK=4)), ("adapters_up", dict(ADAPT, RANK=20)), ("adapters_up", dict(ADAPT, RANK=264)), ("adapters_down", dict(ADAPT, K=4)), ("adapters_down", dict(ADAPT, K=100)),
    ("adapters_down", dict(ADAPT, XT=100)), ("adapters_up", dict(ADAPT, YT=1004)), ("adapters_up", dict(ADAPT, F16=2)), ("adapters_up", dict(ADAPT, N=0)), ("adapters_down", dict(ADAPT, KS=65)),
    ("adapters_up", dict(ADAPT, UT=3)), ("adapters_down", dict(ADAPT, TS=4, RANK=72)), ("adapters_up", dict(ADAPT, UT=1, RANK=72)),
    ("token_logprobs", dict(LOGPROBS, V=0)), ("token_logprobs", dict(LOGPROBS, V=(1 << 19) + 1)), ("token_logprobs", dict(LOGPROBS, TOP=33)), ("token_logprobs", dict(LOGPROBS, V=4, STRIDE=8)),
    ("token_logprobs", dict(LOGPROBS, F16=3)), ("token_logprobs", dict(LOGPROBS, STRIDE=32001)), ("token_logprobs", dict(LOGPROBS, THREADS=100)),
    ("token_logprobs", dict(LOGPROBS, U=17)), ("token_logprobs", dict(LOGPROBS, STRIDE=-8))])
def test_bad_parameters_are_refused(family, params):
    with pytest.raises(_lib.KcgError):
        R.emit_kernel(family, "kernel0", **params)


def test_host_tensors_are_refused_before_anything_is_launched():
    z = torch.zeros
    kc = z(4, 16, 2, 64).to(torch.float8_e4m3fn)
    for call in (lambda: ops.cache_append(z(1, 2, 64), z(1, 2, 64), z(1, 2, 64), kc, kc, z(4, 2), z(4, 2), z(1).long(), z(1).int(), z(5, 64)),
                 lambda: ops.add_adapters(z(1, 8).half(), z(1, 8).half(), z(1, 8, 8).half(), z(1, 8, 8).half(), z(1).int()), lambda: ops.token_logprobs(z(1, 8), z(1).long())):
        with pytest.raises(ValueError):
            call()
