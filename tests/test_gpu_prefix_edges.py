"""The shared prefix (``ops.prefix_decode``) where its parts can go wrong, against float64: sequences a little shorter
than a long prefix, whose own tokens are many parts."""
import pytest
import torch

from test_gpu_prefix import build, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("preset,layout,dtype", [("4bit", "soa", torch.bfloat16), ("3bit", "aos", torch.float16), ("k8v4", "soa", torch.float16)])
@pytest.mark.parametrize("short", [[4095], [0, 4080, 17, 3000, 4095], [4095] * 5])
def test_long_sequences_below_the_prefix(dev, preset, layout, dtype, short):
    lens = [4096, 4100, *short, 4196, 4097]
    check(dev, build(12, lens, 4096, 2, 4, preset=preset, layout=layout, dtype=dtype), 16, sinks=len(short) == 5)
