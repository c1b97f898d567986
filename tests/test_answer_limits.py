"""Where the kernels for adapters and log probabilities read, and what is refused, without a GPU."""
import re
import subprocess

import pytest
import torch

from kernelcodegen_amd import ops, runtime as R
from test_decode_limits import Emitted, Operand


def test_adapters_read_no_column_behind_the_last(tmp_path):
    """The numbers of b that the lanes of adapters_up ask for, by the kernel's own expression, in every pass over the columns: for each rank, tile and type of the
    results that are accepted, with columns that are a whole number of a workgroup's and others."""
    source, names = ["#include <cstdio>", "typedef long long index;"], []
    for rank in range(8, 257, 8):
        for ut in (1, 2, 4):
            if 4 // ut * rank > 256:
                continue
            for f32 in (0, 1):
                step = 4 // ut * (64 if f32 else 128)
                for n in (1, 7, step - 1, step, step + 8, 2 * step, 3 * step - 4, 3 * step):
                    text, _ = R.emit_kernel("adapters_up", "kernel0", N=n, K=64, RANK=rank, F16=0, Y_F32=f32, XT=64, YT=n, ZT=n, UT=ut)
                    # (of names that both launches define, the last is adapters_up's)
                    macros = dict(re.findall(r"^#define (AD_\w+) (.*?)(?: *//.*)?$", text, re.M))
                    where, at = re.search(r"(const int u = [^;]*;)\s*w\[c\] = \*\(const kcg_u32x4\*\)\(b \+ \((.*)\)\);\n", text).groups()
                    names.append("at_%d_%d_%d_%d" % (rank, ut, f32, n))
                    source += ["#define %s %s" % item for item in macros.items()]
                    source.append("""int %s() {
  for (int nb = 0; nb < AD_N; nb += AD_STEP)
    for (int c = 0; c < AD_LOADS; ++c)
      for (int lane = 0; lane < 256; ++lane) {
        struct { int x; } threadIdx = {lane};
        %s
        const index at = %s;
        if (at < 0 || at + 8 > (index)AD_N * AD_RANK) return 1;
      }
  return AD_STEP != %d;
}""" % (names[-1], where, at, step))
                    source += ["#undef " + name for name in macros]
    source.append("int main() {\n%s\n}" % "\n".join('  if (%s()) puts("%s");' % (name, name) for name in names))
    (tmp_path / "reads.cc").write_text("\n".join(source))
    subprocess.check_call(["g++", "-O1", "-w", "-o", str(tmp_path / "reads"), str(tmp_path / "reads.cc")])
    assert len(names) > 800 and subprocess.check_output([str(tmp_path / "reads")], text=True) == ""


def asked_kernels(monkeypatch, tokens, n, k=256, rank=16, adapters=4, inplace=False, f32=False, **cfg):
    """(family, parameters) of the kernels that a call of add_adapters asks for."""
    asked = []

    class Kernel:
        def bind(self, grid):
            return lambda *values: None

    def get_kernel(family, **params):
        asked.append((family, params))
        return Kernel()
    monkeypatch.setattr(R, "get_kernel", get_kernel)
    bf16, i32 = torch.bfloat16, torch.int32
    ops._add_adapters_launch(Operand((tokens, n), torch.float32 if f32 else bf16), Operand((tokens, k), bf16), Operand((adapters, rank, k), bf16),
                             Operand((adapters, n, rank), bf16), Operand((tokens,), i32), Operand((adapters,), torch.float32), inplace, cfg)
    return asked


def test_adapters_kernels_have_only_the_parameters_that_they_depend_on(monkeypatch):
    """Projections that share what they read share the first launch's kernel; the second's does not depend on k."""
    first = [asked_kernels(monkeypatch, 40, n, inplace=inplace, f32=f32)[0] for n, inplace, f32 in ((512, False, False), (1000, False, False), (512, True, False), (512, False, True))]
    assert all(kernel == first[0] for kernel in first) and first[0][0] == "adapters_down"
    second = [asked_kernels(monkeypatch, 40, 512, k)[1] for k in (256, 264, 504)]
    assert all(kernel == second[0] for kernel in second) and second[0][0] == "adapters_up"
    for family, params in (first[0], second[0]):
        text = R.emit_kernel(family, "kernel0", **params)[0]
        for key in params:
            with_other = R.emit_kernel(family, "kernel0", **{**params, key: {"K": 1024, "XT": 1024, "N": 1024, "YT": 1024, "ZT": 1024, "RANK": 32, "KS": 2, "TS": 2, "UT": 2}.get(key, 1 - params[key])})[0]
            assert with_other != text, key
        others = dict(N=77, K=512, XT=512, YT=72, ZT=64, Y_F32=1, SCALES=0, INPLACE=1, ONCE=0, TS=4, UT=4)
        assert R.emit_kernel(family, "kernel0", **{**others, **params})[0] == text


def refused_from(monkeypatch, launch, first):
    """`launch(n)` asks for a kernel below `first` and is refused from there on."""
    def get_kernel(family, **params):
        raise Emitted(params)
    monkeypatch.setattr(R, "get_kernel", get_kernel)
    with pytest.raises(Emitted):
        launch(first - 1)
    for n in (first, 4 * first, 1 << 33):
        with pytest.raises(ValueError):
            launch(n)


def test_a_launch_has_fewer_than_2_to_the_32_threads(monkeypatch):
    bf16, f32, i32, i64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
    for v, threads in ((8, 128), (1 << 18, 512)):            # (a row's workgroup)
        refused_from(monkeypatch, lambda rows: ops._token_logprobs_launch(Operand((rows, v), bf16), Operand((rows,), i64), 0, {}), (1 << 32) // threads)
    refused_from(monkeypatch, lambda rows: ops._token_logprobs_launch(Operand((rows, 4096), f32), Operand((rows,), i64), 5, dict(PARTS=4, THREADS=256)), 1 << 22)
    # the first launch has a workgroup of 256 for 16 tokens; the second, here, one for 64 tokens and 128 columns
    adapters = lambda n: lambda tokens: ops._add_adapters_launch(Operand((tokens, n), bf16), Operand((tokens, 8), bf16), Operand((2, 8, 8), bf16), Operand((2, n, 8), bf16),
                                                                 Operand((tokens,), i32), None, False, dict(NS=16))
    refused_from(monkeypatch, adapters(8), (1 << 28) - 15)
    refused_from(monkeypatch, adapters(2048), (1 << 26) - 63)
    cache, scale = Operand((4, 16, 8, 64), torch.float8_e4m3fn), Operand((4, 8), f32)
    # a wavefront for 16 tokens and a head of the keys or values, and for 32 heads of a token's queries
    refused_from(monkeypatch, lambda tokens: ops._cache_append_launch(Operand((tokens, 32, 64), bf16), Operand((tokens, 8, 64), bf16), Operand((tokens, 8, 64), bf16), cache, cache,
                                                                      scale, scale, Operand((tokens,), i64), Operand((tokens,), i32), Operand((100, 64), f32), False), (1 << 25) - 3)


def test_adapters_parts_of_k_by_columns_and_k():
    """From rank 64 on four parts of k turn into two where the second launch reads them too often, and are no more than k or the part has room for."""
    def parts(tokens, adapters, n, k, rank):
        return ops._add_adapters_form(tokens, adapters, n, k, rank, 128)["KS"]
    for rank in (64, 128):
        assert [parts(64, 64, 4096, k, rank) for k in (2048, 4096, 4104, 11008)] == [2, 2, 4, 4]
        assert [parts(64, 64, n, 4096, rank) for n in (1024, 4088, 4096, 11008)] == [4, 4, 2, 2]
        assert parts(128, 64, 4096, 11008, rank) == 2 and parts(5000, 3, 4096, 11008, rank) <= 4
    assert parts(64, 64, 11008, 4096, 56) == 4
    assert [parts(1, 1, 4096, k, 16) for k in (8, 1024, 1536, 2048, 11008)] == [1, 2, 2, 4, 4]
