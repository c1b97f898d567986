"""The operators of a decoding step at the limits of their arithmetic, against the formulas in 64 bits."""
import math

import pytest
import torch

from kernelcodegen_amd import ops
from test_gpu_decode_step import attention_case, close, ints, plain_attention

pytestmark = pytest.mark.gpu


def again(call):
    """The result of the second of two calls, whose memory is that of the first one's, filled with NaN."""
    call()
    first = call()
    where = first.data_ptr()
    first.fill_(math.nan)
    del first
    second = call()
    assert second.data_ptr() == where
    return second


@pytest.mark.parametrize("d", [32, 96, 128, 160, 224])
@pytest.mark.parametrize("waves,rb", [(1, 1), (1, 2), (2, 1), (2, 2)])
def test_tiles_of_fewer_wavefronts_are_joined_whole(d, waves, rb):
    lengths, counts = [900, 300], [40, 70]
    q, caches, scales, table, starts = attention_case(d + waves, lengths, counts, 4, 2, d, 16, "tokens", "bf16")
    want = plain_attention(q, *caches, *scales, table, lengths, starts, d ** -0.5, 0.0, 0, None)
    keys, first = ints(lengths), ints(starts)
    close(again(lambda: ops.cache_attention(q, *caches, *scales, table, keys, first, SHARE=1, WHOLE=0, WAVES=waves, RB=rb, GRID=50)), want)
