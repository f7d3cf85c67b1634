"""Launch tables of grouped kernels (csrc/devtable.h) that are first met inside a
hipGraph capture: there is room for them wherever the arena stands."""
import pytest
import torch

from distributed_kfac_pytorch_amd.ops.mixed import BF16Weights

pytestmark = pytest.mark.gpu


def test_captures_bring_their_own_tables():
    """64 new tables a capture and 16 between captures, over several arenas of 4 MB."""
    n = 4000
    src = torch.arange(n, device='cuda', dtype=torch.float32)
    dst = torch.zeros(n, device='cuda', dtype=torch.bfloat16)
    caster = BF16Weights(torch.nn.Module())
    at = iter(range(n - 1))

    def cast(count):
        done = []
        for _ in range(count):
            i = next(at)
            caster._cast([(src[i:i + 1], dst[i:i + 1])], 1)
            done.append(i)
        return done
    for _ in range(48):
        cast(16)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            mine = cast(64)
        dst.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(dst[mine], src[mine].to(torch.bfloat16))
