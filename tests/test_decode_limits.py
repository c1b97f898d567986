"""What the operators of a decoding step refuse and how they keep to 32 bits, without a GPU."""
import pytest
import torch

from kernelcodegen_amd import ops, runtime as R


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


def attention(monkeypatch, tokens, batch, width, page=16, heads=1, kv_heads=1, d=32, starts=False, **cfg):
    """The parameters of the kernel that a call would launch."""
    def get_kernel(family, **params):
        raise Emitted(params)
    monkeypatch.setattr(R, "get_kernel", get_kernel)
    caches = [Operand((4, page, kv_heads, d), torch.float8_e4m3fn)] * 2
    scales = [Operand((4, kv_heads), torch.float32)] * 2
    i32 = torch.int32
    with pytest.raises(Emitted) as asked:
        ops._cache_attention_launch(Operand((tokens, heads, d), torch.bfloat16), *caches, *scales, Operand((batch, width), i32), Operand((batch,), i32),
                                    Operand((batch + 1,), i32) if starts else None, None, 0.0, 0, None, cfg)
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
