"""What the operators of a decoding step refuse and how they keep to 32 bits, without a GPU."""
import subprocess

import pytest
import torch

from kernelcodegen_amd import ops, runtime as R
from test_decode_step import ROOT


class Operand:
    """Stands for a device tensor of any size: what the checks of arguments look at."""
    is_cuda = True

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, "cuda"

    def dim(self):
        return len(self.shape)

    def stride(self, at=None):
        out, run = [], 1
        for n in reversed(self.shape):
            out.insert(0, run)
            run *= n
        return tuple(out) if at is None else out[at]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return 1 << 20

    def element_size(self):
        return torch.empty(0, dtype=self.dtype).element_size()


class Emitted(Exception):
    """A kernel is asked for: the arguments have passed."""


def attention(monkeypatch, tokens, batch, width, page=16, heads=1, kv_heads=1, d=32, starts=False, window=0, **cfg):
    """The parameters of the kernel that a call would launch."""
    def get_kernel(family, **params):
        raise Emitted(params)
    monkeypatch.setattr(R, "get_kernel", get_kernel)
    caches = [Operand((4, page, kv_heads, d), torch.float8_e4m3fn)] * 2
    scales = [Operand((4, kv_heads), torch.float32)] * 2
    i32 = torch.int32
    with pytest.raises(Emitted) as asked:
        ops._cache_attention_launch(Operand((tokens, heads, d), torch.bfloat16), *caches, *scales, Operand((batch, width), i32), Operand((batch,), i32),
                                    Operand((batch + 1,), i32) if starts else None, None, 0.0, window, None, cfg)
    return asked.value.args[0]


# A wavefront reads the pages of steps ahead of its own: up to 95 steps of 32 keys of each of 4 wavefronts, and 16 keys.
AHEAD = 95 * 32 * 4 + 16


@pytest.mark.parametrize("page", [16, 256])
def test_positions_ahead_of_the_last_key_stay_within_32_bits(monkeypatch, page):
    room = (0x7FFFFFFF - AHEAD) // page
    for width in (room + 1, 0x7FFFFF00 // page, 1 << 31):
        with pytest.raises(ValueError):
            attention(monkeypatch, 1, 1, width, page)
    attention(monkeypatch, 1, 1, 0x7FFF0000 // page, page)


@pytest.mark.parametrize("waves", [1, 2, 4])
@pytest.mark.parametrize("rb", [1, 2])
def test_a_join_has_workgroups_for_all_columns(waves, rb):
    for d in range(32, 257, 32):
        params = dict(H=2, D=d, PAGE=16, G=4, F16=0, RB=rb, WAVES=waves, SHARE=1, QT=8 * d, QH=d, SCALE=0.1, STARTS=1)
        params.update(KP=32 * d, KT=2 * d, KH=d, VP=32 * d, VT=2 * d, VH=d)
        info = R.emit_kernel("cache_join", "kernel0", **params)[1]
        assert info["grid"][1] * info["block"][0] // 64 >= rb * waves * d // 16


def test_units_of_all_tiles_have_32_bits(monkeypatch):
    """9 heads to a kv head: a tile of 16 rows has one token, and there are as many tiles as tokens."""
    forms = dict(heads=9, starts=True, SHARE=0, WHOLE=0, WAVES=1, RB=1)
    for tokens, keys in ((60000, 1250000), (1, 0x7FFE0000)):
        units = tokens * (keys // 32 - tokens // 64)              # about: of rows that are the last ones of a request
        if units > 1 << 31:
            with pytest.raises(ValueError):
                attention(monkeypatch, tokens, 1, keys // 16, **forms)
        else:
            attention(monkeypatch, tokens, 1, keys // 16, **forms)
    attention(monkeypatch, 6_200_000, 1, 4, starts=True)


PADDED = r"""
#include <cstdio>
#define __device__
#define __forceinline__ inline
#define __restrict__
%s
// units of the tiles of a request, one after the other
static long long counted(const CaRequest& r, long long& idle) {
  long long sum = 0;
  for (int i = 0; i < ca_tiles(r); ++i) {
    const bool keys = r.length - r.count + (i + 1LL) * ca_tokens(r) > 0;
    sum += ca_units(r, i);
    if (!keys && ca_units(r, i) != 1) return -1;
    idle += !keys;
  }
  return sum;
}
int main() {
  // rows behind the last request, and more rows than keys: a tile that sees no key counts one unit, and the closed sums agree
  const int lengths[] = {0, 1, 63, 64, 500, 6000}, counts[] = {1, 2, 63, 129, 700, 4096, 70000};
  for (int length : lengths)
    for (int count : counts) {
      const CaRequest r = {length, count, 0};
      long long idle = 0, sum = counted(r, idle);
      if (sum < 0 || ca_before(r, ca_tiles(r)) != sum) { printf("%%d rows, %%d keys: %%d, counted %%lld\n", count, length, ca_before(r, ca_tiles(r)), sum); return 1; }
      if (length == 0 && sum != ca_tiles(r)) { puts("rows without keys"); return 1; }
    }
  // padding to 2^31 rows stays within 32 bits
  const CaRequest all = {0, 0x7fff0000, 0};
  if (ca_before(all, ca_tiles(all)) != ca_tiles(all)) { puts("all"); return 1; }
  return 0;
}
"""


@pytest.mark.parametrize("window", [0, 1, 100, 0x7FFFFFFF])
@pytest.mark.parametrize("rows,keys", [(1, 128), (4, 32), (12, 128), (64, 64), (128, 64)])
def test_tiles_without_keys_count_one_unit(tmp_path, window, rows, keys):
    text = open(ROOT + "/kernelcodegen_amd/csrc/backend/kernels/cache_attention.hip").read()
    part = text[text.index("struct CaRequest"):text.index("// Request b; b == B")] + text[text.index("// sum of the whole parts"):text.index("// Sum over the lanes up to")]
    source = tmp_path / "units.cc"
    source.write_text("#define CA_WINDOW %d\n#define CA_TOK %d\n#define CA_UK %d\n" % (window, rows, keys) + PADDED % part)
    exe = str(tmp_path / "units")
    subprocess.run(["g++", "-O1", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover", "-o", exe, str(source)], check=True)
    done = subprocess.run([exe], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr


def test_a_window_of_all_keys_is_none(monkeypatch):
    """Positions of rows before the first key are negative: less a window, they have to stay within 32 bits."""
    for window in (160, 1000, 0x7FFFFFFF, 1 << 40):
        assert attention(monkeypatch, 30, 1, 10, starts=True, window=window)["WINDOW"] == 0
    assert attention(monkeypatch, 30, 1, 10, starts=True, window=159)["WINDOW"] == 159
    for tokens, keys in ((1 << 30, 1 << 30), (1 << 26, 1 << 20)):
        for form in ({}, dict(WHOLE=1, SHARE=0, RB=1, WAVES=1)):
            with pytest.raises(ValueError):
                attention(monkeypatch, tokens, 1, keys // 16, starts=True, window=keys - 1, **form)


def test_rows_of_a_4_bit_product_have_32_bits(monkeypatch):
    def get_kernel(family, **params):
        raise Emitted(params)
    monkeypatch.setattr(R, "get_kernel", get_kernel)
    w, scale = Operand((8, 16), torch.uint8), Operand((8, 1), torch.bfloat16)
    for shape, refused in (((1 << 31, 32), True), ((1 << 16, 1 << 15, 32), True), ((0x7FFFFF01, 32), True), ((0x7FFFFF00, 32), False)):
        with pytest.raises(ValueError if refused else Emitted):
            ops._matmul_q4_launch(Operand(shape, torch.bfloat16), w, scale, None, None, {})


# ---- bound launches

def test_the_number_of_free_pages_asks_for_no_other_launch(monkeypatch):
    """The list of free pages and the table's width are another in every step of a loop that passes parts of tensors."""
    made, got = [], []

    def launch(*args):
        made.append(args)
        return lambda *a: got.append(a)
    monkeypatch.setattr(ops, "_page_slots_launch", launch)
    monkeypatch.setattr(ops, "_bound", {})
    i32 = torch.int32
    lengths, table, free = torch.zeros(3, dtype=i32), torch.zeros((3, 40), dtype=i32), torch.zeros(400, dtype=i32)
    for used in range(0, 400, 4):
        ops.page_slots(lengths, lengths, table[:, :1 + used // 20], free[used:], 16, 3)
    assert len(made) == 1 and [(a[6], a[7], a[8]) for a in got] == [(1 + u // 20, 40, 400 - u) for u in range(0, 400, 4)]
    # what is checked by the first call only is in the key
    for other in (dict(free=free[::2]), dict(free=free.long()), dict(free=free[None]), dict(table=table[:, ::2]), dict(table=table[:2]), dict(table=table.long()),
                  dict(lengths=lengths[:2]), dict(page_size=32), dict(tokens=4)):
        before = len(made)
        ops.page_slots(**{**dict(lengths=lengths, added=lengths, table=table, free=free, page_size=16, tokens=3), **other})
        assert len(made) == before + 1, other


@pytest.mark.parametrize("kind", ["plain", "native"])
def test_signatures_of_rows(kind):
    row_signature = R._plain_row_signature if kind == "plain" else __import__("kernelcodegen_amd._launch", fromlist=["x"]).row_signature
    x = torch.zeros((4, 10))
    assert row_signature(x, None) == row_signature(x[:, :3], None) == row_signature(torch.zeros((4, 20))[:, ::20], None) == row_signature(x[:, :0], None)
    different = [row_signature(*t) for t in ((x,), (x[:3],), (x[:, ::2],), (x[0],), (x[:, 1:],), (x.int(),), (x[None],), (x, x), (x, None), (None,), (torch.zeros(()),))]
    assert len(set(different)) == len(different)


def test_bound_launches_are_no_more_than_some():
    kept = type(ops._bound)()
    for i in range(3 * kept.MOST):
        kept[i] = -i
    assert len(kept) == kept.MOST and kept.get(3 * kept.MOST - 1) == 1 - 3 * kept.MOST and kept.get(0) is None
    kept[3 * kept.MOST - 5] = "again"
    assert len(kept) == kept.MOST and kept.get(2 * kept.MOST) == -2 * kept.MOST
