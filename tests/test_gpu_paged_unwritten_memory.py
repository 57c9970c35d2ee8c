"""Paged attention must not depend on what earlier kernels left in shared memory: every SM's shared memory is
filled with words that read as NaN before each call."""

import pytest
import torch

from _paged_util import attend, make_table, values
from test_gpu_paged_cache import engine, random_cache

pytestmark = pytest.mark.gpu

FILL = r"""
extern "C" __global__ void fill(int* sink) {
  __shared__ volatile int s[12288];  // 48 KB: the CTAs that an SM holds together cover it
  for (int i = threadIdx.x; i < 12288; i += blockDim.x) s[i] = -1;
  __syncthreads();
  if (s[threadIdx.x] == 0) *sink = 1;
}
"""


@pytest.fixture(scope="module")
def fill_shared_memory():
    kernel = torch.cuda._compile_kernel(FILL, "fill")
    sink = torch.zeros(1, dtype=torch.int32, device="cuda")
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return lambda: kernel(grid=(32 * sms, 1, 1), block=(256, 1, 1), args=[sink])


@pytest.mark.parametrize("heads", [(12, 2, 128), (8, 1, 128), (4, 2, 64)], ids=str)
@pytest.mark.parametrize("page", [16, 32, 64])
def test_attention_reads_no_unwritten_shared_memory(fill_shared_memory, heads, page):
    hq, hkv, hd = heads
    eng = engine(heads, "bfloat16")
    for rows in (1, 5, 8, 32):
        for length in (5, 33, 65, 130, 397):
            if rows > length:
                continue
            gen = torch.Generator().manual_seed(rows * 1000 + length)
            table, pages = make_table([length], page, gen)
            cache = random_cache(eng, pages, page, gen)
            q = (torch.randn(rows, hq * hd, generator=gen) * 1.5).to(torch.bfloat16).cuda()
            plan, device_table = eng.paged_plan([rows], [length - rows], page_size=page), table.cuda()
            ref, mag, _ = attend(q.double().cpu().view(rows, hq, hd), values(cache.k.cpu()[0]), values(cache.v.cpu()[0]),
                                 cache.k_scale.cpu()[0].double(), cache.v_scale.cpu()[0].double(), table, [rows],
                                 [length - rows], [length - rows], page, 0, hq, hd ** -0.5)
            torch.cuda.synchronize()
            for _ in range(2):
                fill_shared_memory()
                got = eng.paged_attention(cache, 0, plan, device_table, q).double().cpu().view_as(ref)
                assert torch.isfinite(got).all(), (rows, length)
                # probabilities of 8 bits, scores of fp32 and a result rounded to bf16, as for every call
                assert ((got - ref).abs() <= 2.0 ** -7 * mag).all(), (rows, length)
    assert eng.device_error() == 0
