"""Ranges of weight rows of the gradient on codes: as many as the device's SMs take, no fewer than a range's dy in shared memory wants."""
import pytest
import torch

from eridiffusion_b200.ops import functional as F

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("R,N,K,block,grouped", [(1, 15360, 2560, 64, False), (8, 13824, 5120, 64, False), (12, 5120, 2560, 64, True),
                                                 (3, 40, 96, 32, False), (8, 100000, 16384, 64, False)])
def test_planes_follow_the_device(R, N, K, block, grouped):
    cols = 4 * (64 if block % 64 == 0 else 32)
    blocks = -(-K // cols) * ((R + 1) // 2 if grouped else -(-R // 8))
    want = min(torch.cuda.get_device_properties(0).multi_processor_count // blocks, -(-N // 256))
    assert F.N.require().eri_linear_4bit_planes(R, N, K, block, int(grouped)) == max(want, -(-N // 2048), 1)
