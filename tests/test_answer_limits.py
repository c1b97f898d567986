"""Where the kernels for adapters and log probabilities read, and what is refused, without a GPU."""
import re
import subprocess

from kernelcodegen_amd import runtime as R


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
