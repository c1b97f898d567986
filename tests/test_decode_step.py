"""The kernels of a decoding step without a GPU: every form compiles, bad parameters are refused, and the closed forms by which
workgroups find their share of the attention's work agree with counting."""
import os
import subprocess

import pytest
import torch

from kernelcodegen_amd import _lib, ops, runtime as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def cache(d, heads=2, page=16):
    return dict(H=heads, D=d, PAGE=page, KP=heads * d * page, KT=heads * d, KH=d, VP=heads * d * page, VT=heads * d, VH=d)


def attention(d, **more):
    return {**cache(d), **dict(G=4, RB=1, F16=0, QT=8 * d, QH=d, SCALE=0.1), **more}


WRITE = dict(F16=2, WIN=1, XKT=256, XKH=128, XVT=256, XVH=128)
GOOD = [("cache_join", attention(96, SHARE=1, STARTS=1), 2), ("page_slots", dict(PAGE=16), 14), ("cache_write", dict(cache(128), **WRITE), 9), ("cache_write", dict(cache(96), **{**WRITE, "F16": 0, "WIN": 16}), 9),
        ("cache_read", dict(cache(64), F16=0), 6), ("cache_join", attention(128), 2), ("cache_join", attention(256, RB=2, SHARE=1, STARTS=1, WINDOW=100), 2),
        ("gemm_q4", dict(N=100, K=4096, GROUP=128, F16=0, MB=1), 6), ("gemm_q4", dict(N=4096, K=1088, GROUP=64, F16=1, MB=4, ZERO=1, SCALE_F32=1, OUT_F32=1), 6)]
GOOD += [("cache_attention", attention(d, RB=rb, F16=d // 32 % 2, SHARE=share, STARTS=share), 16) for d in range(32, 257, 32) for rb, share in ((1, 0), (1, 1), (2, 1))]
GOOD += [("cache_attention", attention(128, WHOLE=1, CAP=30.0), 16), ("cache_attention", attention(128, WHOLE=1, STARTS=1, WAVES=1), 16), ("cache_attention", attention(128, STARTS=1, WINDOW=500, SLOPES=1, G=40), 16)]


@pytest.mark.parametrize("family,params,nargs", GOOD)
def test_every_form_compiles_for_gfx950(family, params, nargs):
    text, info = R.emit_kernel(family, "kernel0", **params)
    assert info["name"] == "kernel0" and info["num_args"] == nargs and info["workspace_bytes"] == 0
    assert R.compile_to_code(R.prelude() + text)[:4] == b"\x7fELF"


@pytest.mark.parametrize("family,params", [
    ("page_slots", dict(PAGE=16, BLOCK=100)), ("page_slots", dict()), ("page_slots", dict(PAGE=0)), ("cache_read", dict(cache(48), F16=0)), ("cache_read", dict(cache(288), F16=0)), ("cache_read", dict(cache(64, page=8), F16=0)),
    ("cache_read", dict(cache(64, page=48), F16=0)), ("cache_read", dict(cache(64), F16=3)), ("cache_read", dict(cache(64))), ("cache_read", dict(cache(64), F16=0, KT=8)),
    ("cache_read", dict(cache(64), F16=0, KP=-16)), ("cache_write", dict(cache(128), **{**WRITE, "WIN": 65})), ("cache_write", dict(cache(128), **{**WRITE, "XKT": 4})),
    ("cache_attention", attention(128, RB=3)), ("cache_attention", attention(128, RB=4)), ("cache_attention", attention(128, RB=2)), ("cache_attention", attention(128, WAVES=3)), ("cache_attention", attention(128, G=0)), ("cache_attention", attention(128, QT=4)), ("cache_attention", attention(128, KT=1 << 27)),
    ("cache_attention", attention(128, GRID=0)), ("cache_attention", attention(128, CAP=-1.0)), ("cache_attention", attention(128, CAP=float("nan"))),
    ("cache_attention", attention(128, SCALE=float("inf"))), ("cache_attention", attention(128, WINDOW=-1)), ("cache_attention", attention(128, WHOLE=1, SHARE=1)),
    ("cache_join", attention(128, WHOLE=1)), ("cache_attention", attention(128, F16=2)),
    ("gemm_q4", dict(N=100, K=100, GROUP=50, F16=0, MB=1)), ("gemm_q4", dict(N=100, K=192, GROUP=128, F16=0, MB=1)), ("gemm_q4", dict(N=100, K=192, GROUP=96, F16=0, MB=1)),
    ("gemm_q4", dict(N=0, K=128, GROUP=128, F16=0, MB=1)), ("gemm_q4", dict(N=100, K=128, GROUP=128, F16=0, MB=5)), ("gemm_q4", dict(N=100, K=128, GROUP=128, F16=0, MB=4, WK=16, NT=4))])
def test_bad_parameters_are_refused(family, params):
    with pytest.raises(_lib.KcgError):
        R.emit_kernel(family, "kernel0", **params)


def test_host_tensors_are_refused_before_anything_is_launched():
    z = torch.zeros
    kc = z(4, 16, 2, 64).to(torch.float8_e4m3fn)
    for call in (lambda: ops.cache_attention(z(1, 4, 64).half(), kc, kc, z(4, 2), z(4, 2), z(1, 2).int(), z(1).int()),
                 lambda: ops.cache_write(z(1, 2, 64), z(1, 2, 64), kc, kc, z(4, 2), z(4, 2), z(1).long()), lambda: ops.cache_read(kc, z(4, 2), z(1).long()),
                 lambda: ops.matmul_q4(z(1, 64).half(), z(4, 32).byte(), z(4, 1).half()), lambda: ops.page_slots(z(1).int(), z(1).int(), z(1, 1).int(), z(1).int(), 16, 1)):
        with pytest.raises(ValueError):
            call()


HARNESS = r"""
#include <cstdio>
#include <cstdlib>
#define __device__
#define __forceinline__ inline
#define __restrict__
%s
int main() {
  // requests of all kinds: the units of every tile, counted key by key, and the closed sums of them
  for (int count = 0; count < 400; count += count < 40 ? 1 : 37)
    for (int length = 0; length < 3000; length += length < 300 ? 13 : 411) {
      const CaRequest r = {length, count, 0};
      const int tiles = ca_tiles(r), t = ca_tokens(r);
      if (count == 0) { if (tiles) { puts("tiles of no rows"); return 1; } continue; }
      if (t > CA_TOK || (long long)tiles * t < count || (tiles - 1) * t >= count) { puts("tiles"); return 1; }
      long long sum = 0;
      for (int i = 0; i < tiles; ++i) {
        const int units = ca_units(r, i), low = ca_low(r, i) * CA_UK;
        if (ca_before(r, i) != sum || units < 1) { printf("count %%d length %%d tile %%d: %%d, counted %%lld\n", count, length, i, ca_before(r, i), sum); return 1; }
        sum += units;
        for (int row = i * t; row < (i + 1) * t && row < count; ++row) {
          const int pos = length - count + row;
          const int first = CA_WINDOW && pos - CA_WINDOW + 1 > 0 ? pos - CA_WINDOW + 1 : 0;
          if (pos >= 0 && (first < low || pos >= low + units * CA_UK)) { puts("a key outside of the units"); return 1; }
        }
      }
      if (ca_before(r, tiles) != sum) { puts("all"); return 1; }
    }
  for (int i = 0; i < 20000; ++i) {
    const long long n = rand() %% 50, a = rand() %% 300, b = rand() %% 1000, m = 1 + rand() %% 200;
    long long sum = 0;
    for (long long j = 0; j < n; ++j) sum += (a * j + b) / m;
    if (sum != ca_floor_sum(n, a, b, m)) { puts("floor sum"); return 1; }
  }
  return 0;
}
"""


@pytest.mark.parametrize("window", [0, 1, 100, 1000])
@pytest.mark.parametrize("rows,keys", [(1, 128), (4, 32), (4, 64), (12, 128), (64, 128), (64, 32)])
def test_units_of_tiles_in_closed_form(tmp_path, window, rows, keys):
    text = open(os.path.join(ROOT, "kernelcodegen_amd", "csrc", "backend", "kernels", "cache_attention.hip")).read()
    part = text[text.index("struct CaRequest"):text.index("// Request b; b == B")] + text[text.index("// sum of the whole parts"):text.index("// Sum over the lanes up to")]
    source = tmp_path / "units.cc"
    source.write_text("#define CA_WINDOW %d\n#define CA_TOK %d\n#define CA_UK %d\n" % (window, rows, keys) + HARNESS % part)
    exe = str(tmp_path / "units")
    subprocess.run(["g++", "-O1", "-o", exe, str(source)], check=True)
    done = subprocess.run([exe], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
