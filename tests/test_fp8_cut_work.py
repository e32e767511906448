"""Cut work of the FP8 kernels (csrc/cuda/fp8_stream.cu, fp8_gemm.cu): pieces of a tile leave fp32 sums that the warp which arrives last adds up.

The order of memory between the warps cannot be shown by a run, so its shape in the source is what the first test asks for: one function counts arrivals, and in it a
barrier of the warp stands on both sides of the lane that has the fence."""
import zlib
from pathlib import Path

import pytest
import torch

import machx_inference_engine_b200
from machx_inference_engine_b200 import ops
from machx_inference_engine_b200.ops.weights import from_fp8

CUDA = Path(machx_inference_engine_b200.__file__).parent / "csrc" / "cuda"


def test_arrivals_are_counted_between_two_barriers_of_the_warp():
    head, sep, body = (CUDA / "fp8.cuh").read_text().partition("__device__ __forceinline__ bool warp_arrives_last(")
    assert sep
    body = body[:body.index("\n}\n")]
    first, counted, shuffled = body.index("__syncwarp();"), body.index("atom.add.acq_rel.gpu"), body.index("__shfl_sync(")
    assert first < counted < shuffled < body.rindex("__syncwarp();") < body.index("return")
    for name in ("fp8_stream.cu", "fp8_gemm.cu"):
        text = (CUDA / name).read_text()
        assert "warp_arrives_last(p.tickets" in text and "atom." not in text, name


def gen(*key):
    return torch.Generator().manual_seed(zlib.crc32(repr(key).encode()))


# (the cut kernels at their listed kinds: one row whose blocks every CTA rounds, rows rounded before, tiles in pieces along K)
@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 6144, 4096), (1, 6150, 4100), (8, 28672, 1024), (20, 4096, 4096), (40, 4096, 14336), (100, 1024, 8192), (333, 640, 2880)])
def test_cut_sums_repeat_themselves(M, N, K):
    """Two inputs in turn, so that what a launch left behind is never what the next one wants; nothing waits between."""
    g = gen(M, N, K)
    codes = (torch.randn(N, K, generator=g).clamp(-4, 4) * 112).to(torch.float8_e4m3fn)
    w = from_fp8(codes, (0.5 + torch.rand(-(-N // 128), -(-K // 128), generator=g)) * (K ** -0.5 / 112)).to("cuda:0")
    xs = [torch.randn(M, K, generator=g).to("cuda:0", torch.bfloat16) for _ in range(2)]
    want = [ops.linear(x, w, out_f32=True) for x in xs]
    torch.cuda.synchronize()
    wrong = torch.zeros(2, dtype=torch.int64, device="cuda:0")
    for _ in range(200):
        for i, x in enumerate(xs):
            wrong[i] += (ops.linear(x, w, out_f32=True) != want[i]).sum()
    assert wrong.tolist() == [0, 0] and not torch.equal(*want)
