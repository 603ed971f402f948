"""8-bit products of more 256 x 256 tiles than the device has compute units: a workgroup takes several tiles, one's stores under the next one's
loads."""
import pytest

import test_gpu_serving_i8 as i8

pytestmark = pytest.mark.gpu

# 17 x 18 and 25 x 25 tiles, the last ones partly empty in both directions; 1, 2, 3 and 4 pieces of 128 along K, the last one whole or not
SHAPES = [(4300, 4403, 100), (4300, 4403, 300), (4300, 4404, 512), (6200, 6150, 130), (6145, 6400, 33)]


@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("x,out,bias", [("bf16", "bf16", False), ("f32", "f32", True), ("bf16", "bf16", True)])
def test_linear_of_many_tiles(tiny_model, m, n, k, x, out, bias):
    i8.test_linear_matches_whole_numbers(tiny_model, m, n, k, x, out, bias)
