"""shared_prefix_attention behind a kernel that lets its dependents start early and writes the lists
afterwards, as an engine's own metadata kernel may: the call has to see what that kernel wrote."""
import ctypes
import subprocess

import pytest
import torch

from origami_b200 import build
from test_gpu_shared_prefix import BF16, F16, Batch

pytestmark = pytest.mark.gpu

SOURCE = r"""
#include <cuda_runtime.h>
// Lets the next kernel start, spins for a bounded time, then copies src to dst.
__global__ void late(const int* src, int* dst, int n, long long clocks) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const long long begin = clock64();
  while (clock64() - begin < clocks) {
  }
  for (int i = threadIdx.x; i < n; i += blockDim.x) dst[i] = src[i];
}
extern "C" int late_copy(const int* src, int* dst, int n, int clocks, cudaStream_t stream) {
  if (clocks < 0 || clocks > (1 << 21)) return 1;
  late<<<1, 256, 0, stream>>>(src, dst, n, clocks);
  return cudaGetLastError();
}
"""


@pytest.fixture(scope="module")
def late_copy(tmp_path_factory):
    d = tmp_path_factory.mktemp("late")
    (d / "late.cu").write_text(SOURCE)
    subprocess.run([build.nvcc(), *build.NVCC_FLAGS, "-shared", "-o", str(d / "late.so"), str(d / "late.cu")], check=True)
    fn = ctypes.CDLL(str(d / "late.so")).late_copy
    fn.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]

    def run(src, dst):
        assert fn(src.data_ptr(), dst.data_ptr(), src.numel(), 1 << 20, torch.cuda.current_stream().cuda_stream) == 0

    return run


@pytest.mark.parametrize("new, suffix, prefix, Hq, Hk, D, bs, dtype", [
    ([1, 3, 1], [20, 35, 4], 300, 8, 2, 128, 16, BF16),
    ([1] * 64, [1 + 5 * i for i in range(64)], 2000, 32, 8, 128, 16, BF16),
    ([40, 1, 90], [60, 0, 90], 257, 16, 2, 64, 5, F16),
])
def test_lists_written_by_a_kernel_that_triggers_early(cuda, late_copy, new, suffix, prefix, Hq, Hk, D, bs, dtype):
    x = Batch(cuda, new, suffix, prefix, Hq, Hk, D, bs, dtype, seed=17)
    lse = torch.empty(sum(new), Hq, device=cuda)
    want = x.run(lse=lse)
    x.check(want, lse)
    parts = [x.query_start, x.suffix_lens, x.prefix_blocks, x.suffix_blocks.flatten()]
    right = torch.cat(parts)
    # other lists of the same sizes, as good as those: requests of other lengths, other blocks
    B, T = len(new), sum(new)
    other = torch.cat([torch.tensor([0] + [T] * B, dtype=torch.int32, device=cuda), torch.zeros_like(x.suffix_lens),
                       torch.zeros_like(x.prefix_blocks), torch.zeros_like(parts[3])])
    lists = other.clone()
    start, lens, pre, suf = lists.split([p.numel() for p in parts])
    got_lse, out = torch.empty_like(lse), torch.empty_like(want)
    flags = torch.zeros(1, dtype=torch.int32, device=cuda)
    ws = torch.empty(1 << 26, dtype=torch.uint8, device=cuda)
    call = lambda: x.run(query_start=start, suffix_lens=lens, prefix_blocks=pre, suffix_blocks=suf.view(B, -1), out=out,
                         lse=got_lse, workspace=ws, error_flags=flags)
    def late_call():
        late_copy(right, lists)
        call()

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        late_call()
    for step in (late_call, graph.replay):
        for _ in range(3):
            lists.copy_(other)
            out.zero_()
            got_lse.zero_()
            call()  # with the other lists: nothing of them may be left over
            step()
            assert torch.equal(out, want) and torch.equal(got_lse, lse)
    assert int(flags) == 0
