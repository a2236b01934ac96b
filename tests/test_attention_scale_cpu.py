"""CPU: scales that no 32-bit number holds, or whose product with log2 e does not, are
refused before any launch (they would make every output NaN)."""
import importlib

import pytest

X = 1 << 20   # an aligned address that is never read
BAD = [1e39, -1e39, 3e38, -3e38, 1.8e38, float("inf"), float("-inf"), float("nan")]


@pytest.fixture(scope="module")
def lib():
    return importlib.import_module("10_20_b200._lib").lib()


@pytest.mark.parametrize("scale", BAD)
def test_scale_out_of_range(lib, scale):
    x = X
    assert lib.v1x_latent_attention(x, 2304, 576, x, 64, 576, None, 0, x, 64, 64, None, 2, 4, 576, 512, scale, 1, x, x, x,
                                    1 << 30, None, None) == -1
    assert b"scale" in lib.v1x_last_error()
    assert lib.v1x_prompt_attention(x, 768, 192, x, 512, 128, x, 64, x, 512, 128, x, x, 1, 8, 8, 4, 64, scale, 1, x, x,
                                    None, None) == -1
    assert b"scale" in lib.v1x_last_error()
    assert lib.v1x_kv8_attend(x, 512, 128, x, x, x, x, 4, 2, x, 2, 2, x, 1, 4, scale, 1, x, x, x, 1 << 30, None,
                              None) == -1
    assert b"scale" in lib.v1x_last_error()


@pytest.mark.parametrize("scale", BAD)
def test_python_refuses_the_same(scale):
    import torch
    L, K = (importlib.import_module("10_20_b200." + m) for m in ("latent_attention", "kv8"))
    bf, i32 = torch.bfloat16, lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(ValueError, match="finite"):
        L.attend_slots(torch.zeros((2, 4, 576), dtype=bf), torch.zeros((64, 1, 576), dtype=bf), None, i32(2, 8), scale)
    with pytest.raises(ValueError, match="finite"):
        L.attend_prompt(torch.zeros((8, 4, 128), dtype=bf), torch.zeros((8, 4, 128), dtype=bf), None,
                        torch.zeros((8, 4, 128), dtype=bf), i32(2), scale)
    cache = [torch.zeros((4, 2, 64, 128), dtype=torch.float8_e4m3fn), torch.ones((4, 2))] * 2
    with pytest.raises(ValueError, match="finite"):
        K.attend(torch.zeros((1, 4, 128), dtype=bf), *cache, i32(1, 2), i32(1), scale)
