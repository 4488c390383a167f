"""Every kernel and tile that ops.expert_linear chooses from, against float64, at sizes for which the rule picks that one
(fd_expert_linear_kernel): with and without a gate, gathered and in order, several experts with partial tiles, every type.  A
change of the rule that moves a size to another kernel shows here, so that no kernel goes without a test of its values."""
import math

import pytest
import torch

from facedetection_amd import _lib
from test_gpu_expert_block import _close, _gen, _linear64, _routing

pytestmark = pytest.mark.gpu

# kernel, bits of the type, T, k, E, K, N, activation, gated, bias, gather
CASES = [
    ("stream 16 rows, 4 waves", 32, 11, 1, 2, 77, 27, None, False, True, True),
    ("stream 16 rows, 4 waves", 16, 14, 1, 2, 152, 25, "relu", False, True, True),
    ("stream 16 rows, 4 waves", 32, 16, 2, 2, 75, 25, "silu", False, False, False),
    ("stream 16 rows, 4 waves", 16, 11, 1, 2, 160, 25, "gelu", False, True, False),
    ("stream 16 rows, 4 waves", 32, 11, 1, 2, 80, 25, None, True, True, True),
    ("stream 16 rows, 4 waves", 16, 11, 1, 2, 152, 30, "relu", True, False, True),
    ("stream 16 rows, 4 waves", 32, 11, 1, 2, 80, 27, "silu", True, True, False),
    ("stream 16 rows, 4 waves", 16, 16, 1, 2, 152, 28, "gelu", True, True, False),
    ("stream 16 rows, 8 waves", 32, 10, 1, 2, 2382, 25, None, False, False, True),
    ("stream 16 rows, 8 waves", 16, 19, 1, 2, 4131, 25, "relu", False, True, True),
    ("stream 16 rows, 8 waves", 32, 19, 1, 2, 2064, 26, "silu", False, True, False),
    ("stream 16 rows, 8 waves", 16, 14, 1, 2, 4184, 26, "gelu", False, False, False),
    ("stream 16 rows, 8 waves", 32, 17, 1, 2, 2091, 25, None, True, True, True),
    ("stream 16 rows, 8 waves", 16, 12, 1, 2, 4304, 25, "relu", True, True, True),
    ("stream 16 rows, 8 waves", 32, 22, 1, 2, 2128, 26, "silu", True, False, False),
    ("stream 16 rows, 8 waves", 16, 11, 1, 2, 4136, 27, "gelu", True, True, False),
    ("stream 32 rows, 4 waves", 32, 6763, 1, 2, 196, 27, None, False, True, True),
    ("stream 32 rows, 4 waves", 16, 2047, 2, 5, 264, 65, "relu", False, False, True),
    ("stream 32 rows, 4 waves", 32, 4911, 1, 3, 197, 34, "silu", False, True, False),
    ("stream 32 rows, 4 waves", 16, 1941, 1, 3, 840, 50, "gelu", False, True, False),
    ("stream 32 rows, 4 waves", 32, 2045, 2, 3, 100, 38, None, True, False, True),
    ("stream 32 rows, 4 waves", 16, 4470, 1, 5, 200, 34, "relu", True, True, True),
    ("stream 32 rows, 4 waves", 32, 4826, 1, 3, 104, 33, "silu", True, True, False),
    ("stream 32 rows, 4 waves", 16, 2112, 2, 9, 232, 33, "gelu", True, False, False),
    ("tile 32 x 64", 32, 6421, 1, 5, 160, 35, None, False, True, True), ("tile 32 x 64", 16, 1424, 1, 2, 321, 33, "relu", False, True, True),
    ("tile 32 x 64", 32, 3094, 2, 2, 160, 36, "silu", False, False, False), ("tile 32 x 64", 16, 1477, 1, 5, 329, 35, "gelu", False, True, False),
    ("tile 32 x 64", 32, 3004, 1, 9, 168, 53, None, True, True, True), ("tile 32 x 64", 16, 14, 1, 2, 391, 26, "relu", True, False, True),
    ("tile 32 x 64", 32, 3151, 2, 3, 160, 26, "silu", True, True, False), ("tile 32 x 64", 16, 29, 1, 2, 340, 25, "gelu", True, True, False),
    ("tile 64 x 64", 32, 13896, 2, 5, 162, 28, None, False, False, True), ("tile 64 x 64", 16, 2038, 2, 2, 326, 69, "relu", False, True, True),
    ("tile 64 x 64", 32, 13856, 2, 9, 179, 25, "silu", False, True, False), ("tile 64 x 64", 16, 9174, 1, 2, 353, 25, "gelu", False, False, False),
    ("tile 64 x 64", 32, 13321, 1, 9, 190, 34, None, True, True, True), ("tile 64 x 64", 16, 1977, 2, 17, 386, 33, "relu", True, True, True),
    ("tile 64 x 64", 32, 13443, 1, 9, 169, 34, "silu", True, False, False), ("tile 64 x 64", 16, 2032, 2, 5, 367, 36, "gelu", True, True, False),
    ("tile 128 x 128", 16, 15865, 1, 17, 326, 79, None, False, True, True),
    ("tile 128 x 128", 16, 16077, 1, 17, 367, 68, "relu", False, False, False), ("tile 128 x 128", 16, 8772, 2, 9, 337, 36, "silu", True, True, True),
    ("tile 128 x 128", 16, 8369, 2, 5, 333, 34, "gelu", True, True, False), ("dma 64 x 64", 32, 24996, 1, 9, 160, 26, None, False, False, True),
    ("dma 64 x 64", 16, 8269, 2, 3, 328, 26, "relu", False, True, True), ("dma 64 x 64", 32, 26256, 1, 2, 160, 26, "silu", False, True, False),
    ("dma 64 x 64", 16, 16538, 1, 5, 344, 25, "gelu", False, False, False), ("dma 64 x 64", 32, 12384, 1, 17, 160, 34, None, True, True, True),
    ("dma 64 x 64", 16, 4043, 2, 9, 328, 35, "relu", True, True, True), ("dma 64 x 64", 32, 12301, 1, 3, 168, 33, "silu", True, False, False),
    ("dma 64 x 64", 16, 4119, 2, 5, 336, 38, "gelu", True, True, False), ("dma 64 x 128", 16, 17709, 1, 2, 344, 66, None, False, True, True),
    ("dma 64 x 128", 16, 8518, 2, 2, 328, 75, "relu", False, False, False), ("dma 64 x 128", 16, 16857, 1, 5, 344, 33, "silu", True, True, True),
    ("dma 64 x 128", 16, 8256, 2, 3, 320, 34, "gelu", True, True, False), ("dma 128 x 128", 16, 51399, 1, 3, 336, 65, None, False, False, True),
    ("dma 128 x 128", 16, 51149, 1, 9, 320, 66, "relu", False, True, False), ("dma 128 x 128", 16, 25329, 2, 2, 328, 33, "silu", True, True, True),
    ("dma 128 x 128", 16, 12968, 2, 2, 328, 71, "gelu", True, False, False), ("wide 192 x 256", 16, 18860, 2, 9, 352, 136, None, False, True, True),
    ("wide 192 x 256", 16, 32906, 1, 2, 352, 144, "relu", False, True, False),
    ("wide 192 x 256", 16, 16697, 2, 3, 320, 80, "silu", True, False, True), ("wide 192 x 256", 16, 33189, 1, 3, 352, 72, "gelu", True, True, False),
    ("wide 224 x 256", 16, 47779, 1, 17, 344, 136, None, False, True, True),
    ("wide 224 x 256", 16, 24973, 1, 2, 320, 264, "relu", False, False, False),
    ("wide 224 x 256", 16, 23850, 2, 17, 320, 72, "silu", True, True, True), ("wide 224 x 256", 16, 24799, 1, 2, 360, 136, "gelu", True, True, False),
    ("wide 256 x 256", 16, 29721, 2, 2, 328, 136, None, False, False, True),
    ("wide 256 x 256", 16, 30031, 2, 17, 344, 136, "relu", False, True, False),
    ("wide 256 x 256", 16, 29357, 2, 5, 336, 72, "silu", True, True, True), ("wide 256 x 256", 16, 9841, 2, 2, 328, 264, "gelu", True, False, False),
]
TYPES = {32: [torch.float32], 16: [torch.float16, torch.bfloat16]}


@pytest.mark.parametrize("case,dtype", [(c, t) for c in CASES for t in TYPES[c[1]]],
                         ids=lambda v: "%s, %dx%dx%dx%dx%d" % (v[:1] + v[2:7]) if isinstance(v, tuple) else str(v)[6:])
def test_expert_linear_kernel(case, dtype):
    from facedetection_amd import ops
    kernel, _, T, k, E, K, N, act, gated, has_bias, gather = case
    g = _gen(T + 7 * E + K)
    rows, offsets, _, _ = _routing(g, T, E, k, 0.3, 0.03)
    n, S = 2 * N if gated else N, T * k
    x = torch.randn((T if gather else S, K), generator=g, device="cuda").to(dtype)
    w = (torch.randn((E, n, K), generator=g, device="cuda") / math.sqrt(K)).to(dtype)
    bias = torch.randn((E, n), generator=g, device="cuda").to(dtype) if has_bias else None
    rows = rows if gather else None
    number = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    assert _lib.lib().fd_expert_linear_kernel(x.data_ptr(), number, x.shape[0], K, w.data_ptr(), E, N, rows.data_ptr() if gather else None, S,
                                              int(gated)).decode() == kernel
    y = ops.expert_linear(x, w, offsets, rows=rows, bias=bias, activation=act, gated=gated)
    _close(y, *_linear64(x, w, offsets, rows, bias, act, gated))
    assert bool((y[int(offsets[-1]):] == 0).all())
