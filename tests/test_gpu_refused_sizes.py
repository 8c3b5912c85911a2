"""Sizes that the quantised cache and the token log probabilities refuse are
refused in their own manner, before anything of that size is allocated."""
import pytest

from test_gpu_kv_quant import QuantizedKvCache, raises

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top,kind", [(33, "Unsupported"), (49, "Unsupported"), (51, "Shape"), (10 ** 9, "Shape"),
                                      (10 ** 15, "Shape"), (-1, "Shape"), (-10 ** 15, "Shape")])
def test_alternatives(ctx, top, kind):
    import torch
    from uocr_q8.decoder import token_logprobs_device
    x = torch.zeros((3000, 50), device="cuda")
    raises(kind, lambda: token_logprobs_device(ctx, x, None, top))


@pytest.mark.parametrize("first,count", [(0, 10 ** 15), (0, -1), (3, 6), (-1, 1), (9, 0), (10 ** 15, 1), (0, 2 ** 63 - 1),
                                         (0, -2 ** 63)])
def test_slots(ctx, first, count):
    import torch
    kv = QuantizedKvCache(ctx, 1, 2, 32, 4, 10, 4)
    x = torch.ones((4, 64), device="cuda")
    kv.prefill(0, x, x)
    raises("Shape", lambda: kv.read(0, first, count))
    ctx.sync()
    kv.free()
